// Attention of a batch whose sequences share a prefix (include/w4a16_kv.h): the
// plan, the launches and the joining of their shares. The attending kernels are
// those of w4a16_kv_attn.h.
//
// Mathematics. The softmax over a prefix and a sequence's own slots is that over
// the two apart, joined by their states: with R, l, o of each share s,
//     out = sum_s o_s 2^(R_s - R) / sum_s l_s 2^(R_s - R).
// So the rows of all sequences behind one prefix attend it together, as the rows
// of one long sequence would, and a key or value of the prefix is read once for
// all of them.
#include <hip/hip_runtime.h>

#include <cstdint>
#include <string>

#include "w4a16_hip.h"
#include "w4a16_kv_attn.h"
#include "w4a16_kv_host.h"

namespace w4a16 {

// The shares of an output row joined, by W wavefronts (a workgroup of 256
// threads joins 4 / W rows). Lane s holds share s's state (at most 64): those of
// the prefix first, then the sequence's own. `unit` slots a chunk or tile of the
// launches before, `own_rows` rows a workgroup of the own slots' launch: they give
// the shares that were written.
template <int D, int TYPE, int W>
__global__ void __launch_bounds__(256) join_kernel(const AttnArgs prefix, const AttnArgs own, int prefix_unit,
                                                   int own_unit, int own_rows, int64_t rows) {
    constexpr int E = D / 64;   // dims a lane
    constexpr int F = 4;        // shares of a wavefront in flight
    __shared__ float parts[W][D];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % W, lane = threadIdx.x & 63;
    const int64_t row = blockIdx.x * (int64_t)(4 / W) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) / W;
    if (row >= rows) return;   // W == 1 alone: a wavefront for itself
    const float* part = own.partial + row * own.pitch * D + lane * E;
    float v[F][E];
    auto load = [&](int s0) {
#pragma unroll
        for (int x = 0; x < F; ++x)
#pragma unroll
            for (int e = 0; e < E; ++e) v[x][e] = part[(int64_t)min(s0 + W * x, own.pitch - 1) * D + e];
    };
    // requested before the lengths tell which of them were written
    load(wave);
    float2 state = own.states[row * own.pitch + min(lane, own.pitch - 1)];
    const int64_t bt = row / own.heads;
    const int head = (int)(row - bt * own.heads);
    const int b = (int)(bt / own.tokens), t = (int)(bt - (int64_t)b * own.tokens);
    const Seen seen = seen_of(own, b);
    const int r = t * own.group + head % own.group;
    const int end = seen_end(own, seen, r - r % own_rows, own_rows);
    const int own_count = shares_of((end + own_unit - 1) / own_unit, own.splits, own.least).count;
    const int64_t n = prefix.start[b / prefix.sequences];
    const bool known = n >= 0 && n <= prefix.slots;
    const int prefix_count =
        known ? shares_of((int)((n + prefix_unit - 1) / prefix_unit), prefix.splits, prefix.least).count : 0;
    const int64_t p = seen.start + t;
    const bool padding = t >= seen.count;
    const bool inside = !padding && known && p >= 0 && p < own.slots;
    // what was not written may be anything
    const int s = lane - own.share0;
    if (!inside || !(s < 0 ? lane < prefix_count : s < own_count)) state = make_float2(-__builtin_inff(), 0.0f);
    float o[E] = {};
    const float top = wave_max(state.x);
    const float f = state.x == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(state.x - top);
    if (inside) {
        for (int s0 = wave; s0 < own.pitch; s0 += W * F) {
#pragma unroll
            for (int x = 0; x < F; ++x) {
                const int at = s0 + W * x;
                const bool written = at < own.pitch && (at < own.share0 ? at < prefix_count : at - own.share0 < own_count);
                const float fs = __builtin_bit_cast(
                    float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, f), min(at, own.pitch - 1)));
#pragma unroll
                for (int e = 0; e < E; ++e) o[e] = written ? __builtin_fmaf(v[x][e], fs, o[e]) : o[e];
            }
            if (s0 + W * F < own.pitch) load(s0 + W * F);
        }
    }
    if constexpr (W > 1) {
#pragma unroll
        for (int e = 0; e < E; ++e) parts[wave][lane * E + e] = o[e];
        __syncthreads();
        if (wave != 0) return;
#pragma unroll
        for (int w = 1; w < W; ++w)
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] += parts[w][lane * E + e];
    }
    const float inv = padding ? 0.0f : inside ? 1.0f / wave_sum(state.y * f) : __builtin_nanf("");
    uint16_t* out = own.out + row * D + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e) out[e] = (uint16_t)narrow16<TYPE>(o[e] * inv);
}

}  // namespace w4a16

namespace {

using namespace w4a16;
using w4a16_internal::kv_fail;

// How one side (a prefix, or the sequences' own slots) is launched.
struct SidePlan {
    bool prompt;
    int column_tiles;   // NT of the decode form
    int rows_per;
    int64_t row_tiles;
    int unit;           // slots of a chunk or tile
    int splits, least;
    int threads;
};

constexpr int kMostPrefixShares = 48, kMostOwnShares = 16;

SidePlan plan_side(int64_t batch, int64_t rows, int64_t kv_heads, int64_t slots, int64_t dim, int most_shares) {
    SidePlan p;
    p.prompt = rows > 64;
    p.column_tiles = rows <= 16 ? 1 : rows <= 32 || dim == 256 ? 2 : 4;
    p.rows_per = p.prompt ? 128 : 16 * p.column_tiles;
    p.row_tiles = (rows + p.rows_per - 1) / p.rows_per;
    p.unit = p.prompt ? (dim == 256 ? 32 : 64) : 16 * chunk_tiles((int)dim, p.column_tiles);
    p.least = p.prompt ? 2 : 4;
    p.threads = p.prompt && dim <= 128 ? 512 : 256;
    const int64_t groups = batch * kv_heads * p.row_tiles;
    int64_t splits = groups > 0 ? 256 / groups : 1;
    const int64_t most = shares_of((int)((slots + p.unit - 1) / p.unit), most_shares, p.least).count;
    if (splits > most) splits = most;
    p.splits = splits < 1 ? 1 : (int)splits;
    return p;
}

struct Plan {
    SidePlan prefix, own;
    int pitch;
};

Plan plan_shared(int64_t groups, int64_t prefix_slots, int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads,
                 int64_t slots, int64_t dim) {
    const int64_t group = heads / kv_heads;
    Plan p;
    p.prefix = plan_side(groups, batch / groups * tokens * group, kv_heads, prefix_slots, dim, kMostPrefixShares);
    p.own = plan_side(batch, tokens * group, kv_heads, slots, dim, kMostOwnShares);
    p.pitch = p.prefix.splits + p.own.splits;
    return p;
}

template <int D, int CODES, int TYPE, Mode MODE>
void launch_side(const SidePlan& p, const AttnArgs& a, int64_t grid, hipStream_t st) {
    const dim3 g((unsigned)grid), threads((unsigned)p.threads);
    if (p.prompt)
        hipLaunchKernelGGL((prompt_kernel<D, 4, D == 256 ? 1 : 2, CODES, TYPE, MODE>), g, threads, 0, st, a);
    else if (p.column_tiles == 1)
        hipLaunchKernelGGL((decode_kernel<D, 1, CODES, TYPE, MODE>), g, threads, 0, st, a);
    else if (p.column_tiles == 2)
        hipLaunchKernelGGL((decode_kernel<D, 2, CODES, TYPE, MODE>), g, threads, 0, st, a);
    else if constexpr (D <= 128)
        hipLaunchKernelGGL((decode_kernel<D, 4, CODES, TYPE, MODE>), g, threads, 0, st, a);
}

struct Call {
    Plan plan;
    AttnArgs prefix, own;
    int64_t prefix_grid, own_grid, rows;
    hipStream_t stream;
};

template <int D, int CODES, int TYPE>
void launch(const Call& c) {
    launch_side<D, CODES, TYPE, Prefix>(c.plan.prefix, c.prefix, c.prefix_grid, c.stream);
    launch_side<D, CODES, TYPE, Own>(c.plan.own, c.own, c.own_grid, c.stream);
    if (c.plan.pitch > 8)
        hipLaunchKernelGGL((join_kernel<D, TYPE, 4>), dim3((unsigned)c.rows), dim3(256), 0, c.stream, c.prefix, c.own,
                           c.plan.prefix.unit, c.plan.own.unit, c.plan.own.rows_per, c.rows);
    else
        hipLaunchKernelGGL((join_kernel<D, TYPE, 1>), dim3((unsigned)((c.rows + 3) / 4)), dim3(256), 0, c.stream,
                           c.prefix, c.own, c.plan.prefix.unit, c.plan.own.unit, c.plan.own.rows_per, c.rows);
}

template <int D>
void launch_dim(const Call& c, int code_type, int type) {
    if (code_type == W4A16_KV_INT8 && type == W4A16_FP16)
        launch<D, W4A16_KV_INT8, W4A16_FP16>(c);
    else if (code_type == W4A16_KV_INT8)
        launch<D, W4A16_KV_INT8, W4A16_BF16>(c);
    else if (type == W4A16_FP16)
        launch<D, W4A16_KV_FP8, W4A16_FP16>(c);
    else
        launch<D, W4A16_KV_FP8, W4A16_BF16>(c);
}

bool sizes_fit(int64_t groups, int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads) {
    return groups >= 1 && batch >= 0 && batch % groups == 0 && tokens >= 0 && heads >= 1 && kv_heads >= 1 &&
           heads % kv_heads == 0 && batch <= (1 << 24) && tokens <= (1 << 24) && heads <= (1 << 16) &&
           (__int128)(batch / groups) * tokens * (heads / kv_heads) <= (1 << 28);
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
    const Plan p = plan_shared(groups, prefix_slots, batch, tokens, heads, kv_heads, slots, head_dim);
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
    Call c{};
    c.plan = plan_shared(groups, prefix->slots, batch, tokens, heads, cache->kv_heads, cache->slots, dim);
    c.rows = batch * tokens * heads;
    if (workspace == nullptr || workspace_bytes < c.rows * c.plan.pitch * (4 * dim + 8))
        return kv_fail(W4A16_ERR_CONFIG, "the workspace is smaller than w4a16_kv_shared_attention_workspace_bytes");
    if ((reinterpret_cast<uintptr_t>(workspace) & 15u) != 0)
        return kv_fail(W4A16_ERR_ALIGNMENT, "the workspace must be 16-byte aligned");
    c.prefix_grid = groups * cache->kv_heads * c.plan.prefix.row_tiles * c.plan.prefix.splits;
    c.own_grid = batch * cache->kv_heads * c.plan.own.row_tiles * c.plan.own.splits;
    if (!w4a16_internal::launch_fits(c.prefix_grid, c.plan.prefix.threads) ||
        !w4a16_internal::launch_fits(c.own_grid, c.plan.own.threads) || !w4a16_internal::launch_fits(c.rows, 256))
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
    set_cache(c.own, *cache);
    set_plan(c.own, c.plan.own, batch, dim);
    c.stream = static_cast<hipStream_t>(stream);
    if (dim == 64)
        launch_dim<64>(c, cache->code_type, type);
    else if (dim == 128)
        launch_dim<128>(c, cache->code_type, type);
    else
        launch_dim<256>(c, cache->code_type, type);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return kv_fail(W4A16_ERR_LAUNCH, std::string("kernel launch failed: ") + hipGetErrorString(e));
    return W4A16_OK;
}

}  // extern "C"
