// Attention over the 8-bit key/value cache (include/w4a16_kv.h): the plan and
// the launches. The kernels are in w4a16_kv_attn.h.
#include <hip/hip_runtime.h>

#include <cstdint>
#include <string>

#include "w4a16_hip.h"
#include "w4a16_kv_attn.h"
#include "w4a16_kv_host.h"

namespace {

using namespace w4a16;
using w4a16_internal::kv_fail;

// How a call is launched: the form, the rows of a workgroup, the shares of the slots.
struct AttnPlan {
    bool prompt;
    int waves, groups;  // W and KS of the prompt form
    int column_tiles;   // NT of the decode form
    int rows_per;
    int64_t row_tiles;
    int unit;           // slots of a chunk or tile
    int splits, least;  // shares of the slots, and the units of the smallest
};

constexpr int kMaxSplits = 64;

AttnPlan plan_attention(int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t slots, int64_t dim) {
    AttnPlan p;
    const int64_t rows = tokens * (heads / kv_heads);
    p.prompt = rows > 64;
    p.column_tiles = rows <= 16 ? 1 : rows <= 32 || dim == 256 ? 2 : 4;
    // Prompts: a workgroup of 256 rows decodes a tile once for twice the rows,
    // two of 128 rows a compute unit do not wait for each other (32/8 heads of
    // 128: 4096 tokens, 512 workgroups of 256 rows 152 against 168 us; 2000
    // tokens, 256 of them, 68 against 58; 32/4 heads of 64, 2048 tokens 51
    // against 40). head_dim 256 has registers for 128 rows only.
    p.waves = dim <= 128 && batch * kv_heads * ((rows + 255) / 256) >= 512 ? 8 : 4;
    p.rows_per = p.prompt ? 32 * p.waves : 16 * p.column_tiles;
    p.row_tiles = (rows + p.rows_per - 1) / p.rows_per;
    // The rules below know the cache's capacity, not the sequences' lengths, which
    // are on the device: a short prompt in a long cache is planned as a long one.
    // It uses one share then, but the merge is launched and returns at once.
    // Shares of the slots, where the rows alone leave the chip empty. Each writes
    // fp32 outputs and all bring the merge's launch (3 us, 5 to 8 with a prompt's
    // rows).
    // Decoding: one workgroup a compute unit (one token over 130000 slots, 8 KV
    // heads of 128: 56 us, with two 58), two with 17 to 32 rows, whose chunks are
    // shorter (20 rows over 131072 slots: 63 us, with one 83).
    // Prompts: from 1024 slots on, to fill the chip once, and twice from 8192 on
    // (100 tokens behind 4000: 8 shares 29 us, one 99; but 300 tokens from the
    // start 15 us in one share, 20 in two, so shares are of 512 slots at least,
    // 2048 where the rows give more than 64 workgroups).
    const int64_t groups = batch * kv_heads * p.row_tiles;
    p.least = !p.prompt ? 4 : groups <= 64 ? 8 : 32;
    p.unit = p.prompt ? (dim == 256 ? 32 : 64) : 16 * chunk_tiles((int)dim, p.column_tiles);
    int64_t splits = 1;
    if (groups > 0 && p.prompt)
        splits = slots < 1024 ? 1 : (slots < 8192 ? 256 : 512) / groups;
    else if (groups > 0)
        splits = ((p.column_tiles == 2 ? 512 : 256) + groups - 1) / groups;
    const int64_t most = shares_of((int)((slots + p.unit - 1) / p.unit), kMaxSplits, p.least).count;
    if (splits > most) splits = most;
    p.splits = splits < 1 ? 1 : (int)splits;
    // Two groups of wavefronts on the same rows where the rows give less than two
    // workgroups a compute unit and the slots more than ten tiles (32/8 heads of
    // 128, 1500 tokens: 36 us against 44; 300 tokens 14.8 against 13.6).
    p.groups = dim <= 128 && p.waves == 4 && slots >= 640 && groups * p.splits < 512 ? 2 : 1;
    return p;
}

template <int D, int CODES, int TYPE>
void launch_attention(const AttnPlan& p, const AttnArgs& a, int64_t grid, hipStream_t st) {
    const dim3 g((unsigned)grid);
    if (p.prompt && p.waves == 4 && p.groups == 1)
        hipLaunchKernelGGL((prompt_kernel<D, 4, 1, CODES, TYPE>), g, dim3(256), 0, st, a);
    else if (p.prompt) {
        if constexpr (D <= 128) {
            if (p.groups == 2)
                hipLaunchKernelGGL((prompt_kernel<D, 4, 2, CODES, TYPE>), g, dim3(512), 0, st, a);
            else
                hipLaunchKernelGGL((prompt_kernel<D, 8, 1, CODES, TYPE>), g, dim3(512), 0, st, a);
        }
    }
    else if (p.column_tiles == 1)
        hipLaunchKernelGGL((decode_kernel<D, 1, CODES, TYPE>), g, dim3(64 * kDecodeWaves), 0, st, a);
    else if (p.column_tiles == 2)
        hipLaunchKernelGGL((decode_kernel<D, 2, CODES, TYPE>), g, dim3(64 * kDecodeWaves), 0, st, a);
    else if constexpr (D <= 128)
        hipLaunchKernelGGL((decode_kernel<D, 4, CODES, TYPE>), g, dim3(64 * kDecodeWaves), 0, st, a);
}

template <int D, int TYPE>
void launch_typed(const AttnPlan& p, const AttnArgs& a, int code_type, int64_t grid, int64_t rows, hipStream_t st) {
    if (code_type == W4A16_KV_INT8)
        launch_attention<D, W4A16_KV_INT8, TYPE>(p, a, grid, st);
    else
        launch_attention<D, W4A16_KV_FP8, TYPE>(p, a, grid, st);
    if (a.splits > 1)
        hipLaunchKernelGGL((merge_kernel<D, TYPE>), dim3((unsigned)rows), dim3(256), 0, st, a, p.rows_per,
                           p.unit);
}

template <int D>
void launch_dim(const AttnPlan& p, const AttnArgs& a, int code_type, int type, int64_t grid, int64_t rows,
                hipStream_t st) {
    if (type == W4A16_FP16)
        launch_typed<D, W4A16_FP16>(p, a, code_type, grid, rows, st);
    else
        launch_typed<D, W4A16_BF16>(p, a, code_type, grid, rows, st);
}

bool sizes_fit(int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads) {
    return batch >= 0 && tokens >= 0 && heads >= 1 && kv_heads >= 1 && heads % kv_heads == 0 && batch <= (1 << 24) &&
           tokens <= (1 << 24) && heads <= (1 << 16) && tokens * (heads / kv_heads) <= (1 << 28);
}

}  // namespace

extern "C" {

int64_t w4a16_kv_attention_workspace_bytes(int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads,
                                           int64_t slots, int64_t head_dim) {
    if (!sizes_fit(batch, tokens, heads, kv_heads) || slots < 1 || batch == 0 || tokens == 0) return 0;
    const AttnPlan p = plan_attention(batch, tokens, heads, kv_heads, slots, head_dim);
    return p.splits > 1 ? batch * tokens * heads * p.splits * (4 * head_dim + 8) : 0;
}

int w4a16_kv_attention(const w4a16_kv_rows* q, void* out, int64_t tokens, int64_t heads, const w4a16_kv_cache* cache,
                       const int64_t* start, const int64_t* counts, float scale, int type, void* workspace,
                       int64_t workspace_bytes, void* stream) {
    int rc = w4a16_internal::check_kv_cache(cache);
    if (rc != W4A16_OK) return rc;
    if (type != W4A16_FP16 && type != W4A16_BF16) return kv_fail(W4A16_ERR_CONFIG, "queries must be fp16 or bf16");
    if (tokens < 0 || heads < 1 || heads % cache->kv_heads != 0)
        return kv_fail(W4A16_ERR_SHAPE, "heads must be a positive multiple of the cache's KV heads");
    if (!(scale - scale == 0.0f)) return kv_fail(W4A16_ERR_CONFIG, "scale must be a finite number");
    if (!sizes_fit(cache->batch, tokens, heads, cache->kv_heads))
        return kv_fail(W4A16_ERR_TOO_LARGE, "too many tokens or heads");
    if (cache->batch == 0 || tokens == 0) return W4A16_OK;
    if (q == nullptr || q->data == nullptr || out == nullptr || start == nullptr)
        return kv_fail(W4A16_ERR_NULL, "q, out and start must be non-NULL");
    if ((reinterpret_cast<uintptr_t>(q->data) & 1u) != 0 || (reinterpret_cast<uintptr_t>(out) & 15u) != 0)
        return kv_fail(W4A16_ERR_ALIGNMENT, "q must be 2-byte and out 16-byte aligned");
    const int64_t dim = cache->head_dim, batch = cache->batch;
    const AttnPlan p = plan_attention(batch, tokens, heads, cache->kv_heads, cache->slots, dim);
    const int64_t rows = batch * tokens * heads;
    if (p.splits > 1) {
        if (workspace == nullptr || workspace_bytes < rows * p.splits * (4 * dim + 8))
            return kv_fail(W4A16_ERR_CONFIG, "the workspace is smaller than w4a16_kv_attention_workspace_bytes");
        if ((reinterpret_cast<uintptr_t>(workspace) & 15u) != 0)
            return kv_fail(W4A16_ERR_ALIGNMENT, "the workspace must be 16-byte aligned");
    }
    const int64_t grid = batch * cache->kv_heads * p.row_tiles * p.splits;
    const int threads = 64 * (p.prompt ? p.waves * p.groups : kDecodeWaves);
    if (!w4a16_internal::launch_fits(grid, threads) || rows > 0x7FFFFFFF)
        return kv_fail(W4A16_ERR_TOO_LARGE, "too many rows for one launch");
    AttnArgs a{};
    a.q = static_cast<const uint16_t*>(q->data);
    a.out = static_cast<uint16_t*>(out);
    a.k_codes = static_cast<const uint8_t*>(cache->k.codes);
    a.v_codes = static_cast<const uint8_t*>(cache->v.codes);
    a.k_scales = cache->k.scales;
    a.v_scales = cache->v.scales;
    a.start = start;
    a.counts = counts;
    // the outputs come first, so that both start on 16 bytes
    a.partial = static_cast<float*>(workspace);
    a.states = reinterpret_cast<float2*>(static_cast<float*>(workspace) + (p.splits > 1 ? rows * p.splits * dim : 0));
    a.qb = q->batch_stride;
    a.qt = q->token_stride;
    a.qh = q->head_stride;
    a.kb = cache->k.batch_stride;
    a.kh = cache->k.head_stride;
    a.vb = cache->v.batch_stride;
    a.vh = cache->v.head_stride;
    a.ksb = cache->k.scale_batch_stride;
    a.ksh = cache->k.scale_head_stride;
    a.vsb = cache->v.scale_batch_stride;
    a.vsh = cache->v.scale_head_stride;
    a.slots = cache->slots;
    a.scale = scale;
    a.tokens = (int)tokens;
    a.heads = (int)heads;
    a.kv_heads = (int)cache->kv_heads;
    a.group = (int)(heads / cache->kv_heads);
    a.block_log = cache->block == 16 ? 4 : cache->block == 32 ? 5 : cache->block == 64 ? 6 : 7;
    a.splits = p.splits;
    a.least = p.least;
    // first chunks of up to 8 MB in all (one token over 1500 of 2048 slots, 32/4
    // heads of 64: 7.4 against 8.1 us)
    a.early = batch * cache->kv_heads * p.row_tiles * p.splits * 4 * p.unit * dim * 2 <= (8 << 20);
    a.row_tiles = (int)p.row_tiles;
    a.vec = (reinterpret_cast<uintptr_t>(q->data) & 15u) == 0 &&
            ((q->batch_stride | q->token_stride | q->head_stride) & 7) == 0;
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (dim == 64)
        launch_dim<64>(p, a, cache->code_type, type, grid, rows, st);
    else if (dim == 128)
        launch_dim<128>(p, a, cache->code_type, type, grid, rows, st);
    else
        launch_dim<256>(p, a, cache->code_type, type, grid, rows, st);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return kv_fail(W4A16_ERR_LAUNCH, std::string("kernel launch failed: ") + hipGetErrorString(e));
    return W4A16_OK;
}

}  // extern "C"
