// Attention of a batch whose sequences share a prefix (include/w4a16_kv.h): the
// checks and the plan. The kernels are in w4a16_kv_shared.h.
#include <hip/hip_runtime.h>

#include <cstdint>
#include <string>

#include "w4a16_hip.h"
#include "w4a16_kv_host.h"
#include "w4a16_kv_shared.h"

namespace {

using namespace w4a16;
using w4a16_internal::kv_fail;

constexpr int kMostPrefixShares = 48, kMostOwnShares = 16;

// Rows a workgroup, and the slots' shares: at most `most_shares`, and so many that up to
// `workgroups` are launched, as one more on a compute unit than on the others is waited
// for (42 rows behind each of 3 prefixes of 30001 slots, 8 KV heads of 128: 504 of 512
// workgroups 52 us, 528 67).
SidePlan plan_side(int64_t batch, int64_t rows, int64_t kv_heads, int64_t slots, int64_t dim, int most_shares,
                   int64_t workgroups, SidePlan p) {
    p.rows_per = p.prompt ? 32 * p.waves : 16 * p.column_tiles;
    p.row_tiles = (rows + p.rows_per - 1) / p.rows_per;
    p.unit = p.prompt ? (dim == 256 ? 32 : 64) : 16 * chunk_tiles((int)dim, p.column_tiles);
    p.threads = 64 * (p.prompt ? p.waves : kDecodeWaves);
    const int64_t groups = batch * kv_heads * p.row_tiles;
    int64_t splits = groups > 0 ? workgroups / groups : 1;
    // two fit a compute unit (4 rows behind each of 17 prefixes of 4000 slots: a share 46
    // us, three 39)
    if (splits < 2 && groups <= 256 && p.threads <= 256) splits = groups > 128 ? 512 / groups : 2;
    const int64_t most = shares_of((int)((slots + p.unit - 1) / p.unit), most_shares, p.least).count;
    if (splits > most) splits = most;
    p.splits = splits < 1 ? 1 : (int)splits;
    return p;
}

// Workgroups of a prefix's prompt form, of which a compute unit holds one, for `groups`
// of them a share: the number of shares with the shortest rounds over the chip. In tiles,
// a round takes its share and about 5, a share of 256 workgroups about 8 to write and
// join (32/8 heads of 128, us with 1 to 5 shares: 1200 tokens behind 8000 246, 273, 207,
// 244, 223; 800 behind 3000 103, 72, 97, 90, 94; 2500 behind 6000 393, 337, 325, 341, -).
int64_t prompt_workgroups(int64_t groups, int64_t slots, int64_t dim) {
    const int64_t tiles = (slots + (dim == 256 ? 31 : 63)) / (dim == 256 ? 32 : 64);
    int64_t best = 0, shares = 1;
    for (int64_t s = 1; s <= kMostPrefixShares; ++s) {
        const int64_t cost = 30 * ((groups * s + 255) / 256) * ((tiles + s - 1) / s + 5) + s * groups;
        if (s == 1 || cost < best) {
            best = cost;
            shares = s;
        }
    }
    return groups * shares;
}

SharedPlan plan_shared(int64_t groups, int64_t prefix_slots, int64_t batch, int64_t tokens, int64_t heads,
                       int64_t kv_heads, int64_t slots, int64_t dim) {
    const int64_t group = heads / kv_heads, rows = tokens * group, all = batch / groups * rows;
    SharedPlan p{};
    SidePlan prefix{}, own{};
    prefix.waves = own.waves = 4;
    own.prompt = rows > 64;
    own.column_tiles = rows <= 16 ? 1 : 2;
    // The rules below know the caches' capacities, not the lengths, which are on the device.
    if (own.prompt) {
        // Two launches, the second of which joins the prefix's shares unless its own
        // rows leave the chip empty. Workgroups of 256 rows of the prefix (4 x 500
        // tokens, 32/8 heads of 128, behind 6000: 196 us, of 128 rows 218), of a
        // sequence's own rows as attention over one cache has them (202 with 256).
        prefix.prompt = true;
        prefix.waves = wide_waves((int)dim);
        const bool many = batch * kv_heads * ((rows + 255) / 256) >= 512;
        own.waves = many ? prefix.waves : 4;
        prefix.least = own.least = 8;
        p.prefix = plan_side(groups, all, kv_heads, prefix_slots, dim, kMostPrefixShares,
                             prompt_workgroups(groups * kv_heads * ((all + 32 * prefix.waves - 1) / (32 * prefix.waves)),
                                               prefix_slots, dim),
                             prefix);
        p.own = plan_side(batch, rows, kv_heads, slots, dim, many ? 1 : kMostOwnShares, 256, own);
        p.last = p.own.splits == 1;
    } else {
        // One launch for both, and one that joins. The prefix in the decode form up to 64
        // rows; of 128 dims up to 128 over short prefixes (128 rows over 6000 slots: 22 us,
        // in the prompt form 27; over 8192 slots the other way round); of 64 dims, whose
        // codes are fewer to decode, until the products are many (128 rows over 1500 slots:
        // 10.3 us, in the prompt form 11.8; 256 over 6000: 16.5 and 21; 192 over 50000: 45
        // and 39). 32 rows a workgroup (64 of 64 dims over 8000 slots: 11.7 us, 64 rows a
        // workgroup 14.8), 48 where these are all (42 of 128 dims over 4 x 30001: 41 us, of
        // 32 rows 47). One workgroup a compute unit, two for 17 to 48 rows of 128 dims over
        // long prefixes (32 rows over 100000 slots: 52 us, one 54; 16 rows 53, one 47). In
        // the prompt form, which has the matrix cores to do, fewer workgroups where the
        // sequences' own slots, which have the memory, take as long (64 sequences of up to
        // 1024 slots behind 8192: 160 workgroups 37 us, 256 of them 44; of up to 64 behind
        // 32768: 63, and 128 of them 95; 256 sequences of 8 rows, of up to 256 slots behind
        // 8000: 81, and 256 of them 52). Of 92 sizes (24 to 256 sequences, 2000 to 32768
        // prefix slots, 64 to 4096 own ones, six layouts of heads of 64 to 256 dims), each
        // with 96 to 320 workgroups, these two lie within 10% of the best number for 80; far
        // from it are 24 sequences of 1024 slots behind 8192 (35 us, 160 workgroups 27) and
        // of 4096 (41, 96 of them 34), 24 of 256 dims and 512 slots (55, 160 of them 45).
        prefix.prompt = dim == 64 ? all > 64 && (__int128)all * prefix_slots > (6 << 20)
                                  : all > (dim == 128 && prefix_slots <= 6144 ? 128 : 64);
        prefix.column_tiles = all <= 16 ? 1 : all > 32 && all <= 48 && dim == 128 ? 3 : 2;
        if (prefix.column_tiles < own.column_tiles) prefix.column_tiles = own.column_tiles;
        prefix.least = prefix.prompt ? 2 : 4;
        own.least = 4;
        const bool beside = batch / groups * slots >= 4 * prefix_slots && rows * prefix_slots < 64 * slots;
        const int64_t workgroups = prefix.prompt ? (beside ? 160 : 256)
                                   : prefix.column_tiles >= 2 && all <= 48 && dim == 128 && prefix_slots >= 8192 ? 512 : 256;
        p.prefix = plan_side(groups, all, kv_heads, prefix_slots, dim, kMostPrefixShares, workgroups, prefix);
        p.own = plan_side(batch, rows, kv_heads, slots, dim, kMostOwnShares, 256, own);
    }
    p.pitch = p.prefix.splits + (p.last ? 0 : p.own.splits);
    return p;
}

bool sizes_fit(int64_t groups, int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads) {
    return groups >= 1 && batch >= 0 && batch % groups == 0 && tokens >= 0 && heads >= 1 && kv_heads >= 1 &&
           heads % kv_heads == 0 && batch <= (1 << 24) && tokens <= (1 << 24) && heads <= (1 << 16) &&
           (__int128)(batch / groups) * tokens * (heads / kv_heads) <= (1 << 28) &&
           (__int128)batch * tokens * heads <= ((int64_t)1 << 40);
}

void set_cache(AttnArgs& a, const w4a16_kv_cache& c) {
    a.k_codes = static_cast<const uint8_t*>(c.k.codes);
    a.v_codes = static_cast<const uint8_t*>(c.v.codes);
    a.k_scales = c.k.scales;
    a.v_scales = c.v.scales;
    a.kb = c.k.batch_stride;
    a.kh = c.k.head_stride;
    a.vb = c.v.batch_stride;
    a.vh = c.v.head_stride;
    a.ksb = c.k.scale_batch_stride;
    a.ksh = c.k.scale_head_stride;
    a.vsb = c.v.scale_batch_stride;
    a.vsh = c.v.scale_head_stride;
    a.slots = c.slots;
    a.block_log = c.block == 16 ? 4 : c.block == 32 ? 5 : c.block == 64 ? 6 : 7;
}

void set_plan(AttnArgs& a, const SidePlan& p, int64_t batch, int64_t dim) {
    a.splits = p.splits;
    a.least = p.least;
    a.row_tiles = (int)p.row_tiles;
    // first chunks of up to 8 MB in all
    a.early = batch * a.kv_heads * p.row_tiles * p.splits * 4 * p.unit * dim * 2 <= (8 << 20);
}

}  // namespace

extern "C" {

int64_t w4a16_kv_shared_attention_workspace_bytes(int64_t groups, int64_t prefix_slots, int64_t batch, int64_t tokens,
                                                  int64_t heads, int64_t kv_heads, int64_t slots, int64_t head_dim) {
    if (!sizes_fit(groups, batch, tokens, heads, kv_heads) || prefix_slots < 1 || slots < 1 || batch == 0 || tokens == 0)
        return 0;
    const SharedPlan p = plan_shared(groups, prefix_slots, batch, tokens, heads, kv_heads, slots, head_dim);
    return batch * tokens * heads * p.pitch * (4 * head_dim + 8);
}

int w4a16_kv_shared_attention(const w4a16_kv_rows* q, void* out, int64_t tokens, int64_t heads,
                              const w4a16_kv_cache* prefix, const int64_t* prefix_lengths, const w4a16_kv_cache* cache,
                              const int64_t* start, const int64_t* counts, float scale, int type, void* workspace,
                              int64_t workspace_bytes, void* stream) {
    int rc = w4a16_internal::check_kv_cache(prefix);
    if (rc != W4A16_OK || (rc = w4a16_internal::check_kv_cache(cache)) != W4A16_OK) return rc;
    if (type != W4A16_FP16 && type != W4A16_BF16) return kv_fail(W4A16_ERR_CONFIG, "queries must be fp16 or bf16");
    if (prefix->kv_heads != cache->kv_heads || prefix->head_dim != cache->head_dim ||
        prefix->code_type != cache->code_type)
        return kv_fail(W4A16_ERR_SHAPE, "the prefix and the cache must have the same KV heads, head_dim and codes");
    if (prefix->batch < 1 || cache->batch % prefix->batch != 0)
        return kv_fail(W4A16_ERR_SHAPE, "the cache's sequences must be a multiple of the prefixes");
    if (tokens < 0 || heads < 1 || heads % cache->kv_heads != 0)
        return kv_fail(W4A16_ERR_SHAPE, "heads must be a positive multiple of the cache's KV heads");
    if (!(scale - scale == 0.0f)) return kv_fail(W4A16_ERR_CONFIG, "scale must be a finite number");
    if (!sizes_fit(prefix->batch, cache->batch, tokens, heads, cache->kv_heads))
        return kv_fail(W4A16_ERR_TOO_LARGE, "too many tokens or heads");
    if (cache->batch == 0 || tokens == 0) return W4A16_OK;
    if (q == nullptr || q->data == nullptr || out == nullptr || start == nullptr || prefix_lengths == nullptr)
        return kv_fail(W4A16_ERR_NULL, "q, out, start and the prefixes' lengths must be non-NULL");
    if ((reinterpret_cast<uintptr_t>(q->data) & 1u) != 0 || (reinterpret_cast<uintptr_t>(out) & 15u) != 0)
        return kv_fail(W4A16_ERR_ALIGNMENT, "q must be 2-byte and out 16-byte aligned");
    const int64_t dim = cache->head_dim, batch = cache->batch, groups = prefix->batch;
    SharedCall c{};
    c.plan = plan_shared(groups, prefix->slots, batch, tokens, heads, cache->kv_heads, cache->slots, dim);
    c.rows = batch * tokens * heads;
    if (workspace == nullptr || workspace_bytes < c.rows * c.plan.pitch * (4 * dim + 8))
        return kv_fail(W4A16_ERR_CONFIG, "the workspace is smaller than w4a16_kv_shared_attention_workspace_bytes");
    if ((reinterpret_cast<uintptr_t>(workspace) & 15u) != 0)
        return kv_fail(W4A16_ERR_ALIGNMENT, "the workspace must be 16-byte aligned");
    c.prefix_grid = groups * cache->kv_heads * c.plan.prefix.row_tiles * c.plan.prefix.splits;
    c.own_grid = batch * cache->kv_heads * c.plan.own.row_tiles * c.plan.own.splits;
    if (!w4a16_internal::launch_fits((__int128)c.prefix_grid + c.own_grid, 512) ||
        (!c.plan.last && !w4a16_internal::launch_fits(c.rows, 256)))
        return kv_fail(W4A16_ERR_TOO_LARGE, "too many rows for one launch");
    AttnArgs a{};
    a.q = static_cast<const uint16_t*>(q->data);
    a.out = static_cast<uint16_t*>(out);
    a.counts = counts;
    // the outputs come first, so that both start on 16 bytes
    a.partial = static_cast<float*>(workspace);
    a.states = reinterpret_cast<float2*>(static_cast<float*>(workspace) + c.rows * c.plan.pitch * dim);
    a.qb = q->batch_stride;
    a.qt = q->token_stride;
    a.qh = q->head_stride;
    a.scale = scale;
    a.heads = (int)heads;
    a.kv_heads = (int)cache->kv_heads;
    a.group = (int)(heads / cache->kv_heads);
    a.vec = (reinterpret_cast<uintptr_t>(q->data) & 15u) == 0 &&
            ((q->batch_stride | q->token_stride | q->head_stride) & 7) == 0;
    a.pitch = c.plan.pitch;
    a.sequences = (int)(batch / groups);
    a.sequence_tokens = (int)tokens;
    c.prefix = c.own = a;
    c.prefix.start = prefix_lengths;
    c.prefix.tokens = (int)(batch / groups * tokens);
    set_cache(c.prefix, *prefix);
    set_plan(c.prefix, c.plan.prefix, groups, dim);
    c.own.start = start;
    c.own.tokens = (int)tokens;
    c.own.share0 = c.plan.prefix.splits;
    c.own.prefix_lengths = prefix_lengths;
    c.own.prefix_slots = prefix->slots;
    c.own.prefix_unit = c.plan.prefix.unit;
    c.own.prefix_splits = c.plan.prefix.splits;
    c.own.prefix_least = c.plan.prefix.least;
    set_cache(c.own, *cache);
    set_plan(c.own, c.plan.own, batch, dim);
    c.stream = static_cast<hipStream_t>(stream);
    if (dim == 64)
        launch_shared<64>(c, cache->code_type, type);
    else if (dim == 128)
        launch_shared<128>(c, cache->code_type, type);
    else
        launch_shared<256>(c, cache->code_type, type);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return kv_fail(W4A16_ERR_LAUNCH, std::string("kernel launch failed: ") + hipGetErrorString(e));
    return W4A16_OK;
}

}  // extern "C"
