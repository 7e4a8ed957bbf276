// Copying sequences from one 8-bit cache to another, and moving them within one
// (include/w4a16_kv.h). Codes and scales are copied as they are.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <string>

#include "w4a16_hip.h"
#include "w4a16_kv_device.h"
#include "w4a16_kv_host.h"

namespace w4a16 {

struct MoveSide {
    const uint8_t* from;
    uint8_t* to;
    const float* from_scales;
    float* to_scales;
    int64_t fb, fh, tb, th, fsb, fsh, tsb, tsh;
};

struct MoveArgs {
    MoveSide side[2];
    const int64_t *source, *lengths;
    int64_t slots;                  // that both caches have
    int batch, held, kv_heads;      // sequences written, and read from
    int units, block_log;           // 16-byte units of a slot
    int chunk, chunks;              // slots of a workgroup
};

// Slots of sequence b's source that are copied; 0 where it has none.
__device__ __forceinline__ int64_t moved_slots(const MoveArgs& a, int64_t source) {
    return source < 0 || source >= a.held ? 0 : min(max(a.lengths[source], (int64_t)0), a.slots);
}

// A store of 16 bytes; past the caches where much is moved.
template <bool FAR>
__device__ __forceinline__ void put(u32x4* to, u32x4 v) {
    if constexpr (FAR)
        __builtin_nontemporal_store(v, to);
    else
        *to = v;
}

// ---------------------------------------------------------------------------
// Between two caches: a workgroup copies a chunk of a head of one sequence, 16
// bytes a lane and load, the blocks that start in it with their scales.
//
// Bound: memory (3 sequences of up to 4001 tokens, 8 KV heads of 128, into 24: 30
// us for 91 MB written; 61 with the sequences of a chunk one after the other and
// stores that stay in the caches, 40 and 50 with one of the two).
// ---------------------------------------------------------------------------
constexpr int kForkUnits = 2;   // of a thread: 30 us, with four 32, with one 51

template <bool FAR>
__global__ void __launch_bounds__(256) fork_kernel(const MoveArgs a) {
    int item = blockIdx.x;
    const int64_t slot0 = (int64_t)(item % a.chunks) * a.chunk;
    item /= a.chunks;
    const int h = item % a.kv_heads;
    item /= a.kv_heads;
    const MoveSide& s = a.side[item & 1];
    const int b = item >> 1;
    const int64_t source = a.source[b];
    const int64_t slots = moved_slots(a, source);
    if (slot0 >= slots) return;
    const int n = (int)min((int64_t)a.chunk, slots - slot0);
    const u32x4* from = reinterpret_cast<const u32x4*>(s.from + source * s.fb + h * s.fh) + slot0 * a.units;
    u32x4* to = reinterpret_cast<u32x4*>(s.to + b * s.tb + h * s.th) + slot0 * a.units;
    u32x4 v[kForkUnits];
#pragma unroll
    for (int i = 0; i < kForkUnits; ++i) {
        const int u = (int)threadIdx.x + 256 * i;
        if (u < n * a.units) v[i] = from[u];
    }
    const int64_t block = ((slot0 + (1 << a.block_log) - 1) >> a.block_log) + threadIdx.x;
    if (block << a.block_log < slot0 + n)
        s.to_scales[b * s.tsb + h * s.tsh + block] = s.from_scales[source * s.fsb + h * s.fsh + block];
#pragma unroll
    for (int i = 0; i < kForkUnits; ++i) {
        const int u = (int)threadIdx.x + 256 * i;
        if (u < n * a.units) put<FAR>(to + u, v[i]);
    }
}

// ---------------------------------------------------------------------------
// Within a cache: a workgroup holds the same slots of a head of all sequences in
// registers, U units a thread, and writes none before all are read.
//
// Bound: memory (beams of 32 sequences of up to 2000 tokens, 8 KV heads of 128: 33
// us for 75 MB written; 51 with stores that stay in the caches, 60 with 16 units a
// thread).
// ---------------------------------------------------------------------------
template <int T, int U, bool FAR>
__global__ void __launch_bounds__(T) reorder_kernel(const MoveArgs a) {
    int item = blockIdx.x;
    const int h = item % a.kv_heads;
    item /= a.kv_heads;
    const MoveSide& s = a.side[item & 1];
    const int64_t slot0 = (int64_t)(item >> 1) * a.chunk;
    const int row = a.chunk * a.units;   // units of a sequence
    // scales of the blocks that start here, `starts` of a sequence
    const int64_t block0 = (slot0 + (1 << a.block_log) - 1) >> a.block_log;
    const int64_t end = min(slot0 + a.chunk, a.slots);
    const int starts = (int)max(((end + (1 << a.block_log) - 1) >> a.block_log) - block0, (int64_t)0);
    constexpr int S = U / 4;   // 4 units a slot at least, and a block has 16 slots
    u32x4 v[U];
    float scale[S];
    bool moves[U], scale_moves[S];
#pragma unroll
    for (int i = 0; i < U; ++i) {
        const int u = (int)threadIdx.x + T * i;
        const int b = u / row, at = u - b * row;
        moves[i] = false;
        if (b < a.batch) {
            const int64_t source = a.source[b];
            moves[i] = source != b && slot0 + at / a.units < moved_slots(a, source);
            if (moves[i])
                v[i] = reinterpret_cast<const u32x4*>(s.to + source * s.tb + h * s.th)[slot0 * a.units + at];
        }
    }
#pragma unroll
    for (int i = 0; i < S; ++i) {
        const int u = (int)threadIdx.x + T * i;
        scale_moves[i] = false;
        if (u < a.batch * starts) {
            const int b = u / starts;
            const int64_t source = a.source[b], block = block0 + u - b * starts;
            scale_moves[i] = source != b && block << a.block_log < moved_slots(a, source);
            if (scale_moves[i]) scale[i] = s.to_scales[source * s.tsb + h * s.tsh + block];
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // every load has returned before any store of the workgroup
    __syncthreads();
#pragma unroll
    for (int i = 0; i < U; ++i) {
        const int u = (int)threadIdx.x + T * i;
        const int b = u / row, at = u - b * row;
        if (moves[i]) put<FAR>(reinterpret_cast<u32x4*>(s.to + b * s.tb + h * s.th) + slot0 * a.units + at, v[i]);
    }
#pragma unroll
    for (int i = 0; i < S; ++i) {
        const int u = (int)threadIdx.x + T * i;
        if (!scale_moves[i]) continue;
        const int b = u / starts;
        s.to_scales[b * s.tsb + h * s.tsh + block0 + u - b * starts] = scale[i];
    }
}

}  // namespace w4a16

namespace {

using namespace w4a16;
using w4a16_internal::kv_fail;

MoveSide side_of(const w4a16_kv_codes& from, const w4a16_kv_codes& to) {
    return {static_cast<const uint8_t*>(from.codes), static_cast<uint8_t*>(to.codes), from.scales, to.scales,
            from.batch_stride, from.head_stride, to.batch_stride, to.head_stride, from.scale_batch_stride,
            from.scale_head_stride, to.scale_batch_stride, to.scale_head_stride};
}

MoveArgs args_of(const w4a16_kv_cache& from, const w4a16_kv_cache& to, const int64_t* source, const int64_t* lengths) {
    MoveArgs a{};
    a.side[0] = side_of(from.k, to.k);
    a.side[1] = side_of(from.v, to.v);
    a.source = source;
    a.lengths = lengths;
    a.slots = std::min(from.slots, to.slots);
    a.batch = (int)to.batch;
    a.held = (int)from.batch;
    a.kv_heads = (int)to.kv_heads;
    a.units = (int)(to.head_dim / 16);
    a.block_log = to.block == 16 ? 4 : to.block == 32 ? 5 : to.block == 64 ? 6 : 7;
    return a;
}

// Whether a cache is too large to stay in the device's caches between calls.
bool is_far(const w4a16_kv_cache& c) {
    return (__int128)2 * c.batch * c.kv_heads * c.slots * c.head_dim > (32 << 20);
}

int finish() {
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return kv_fail(W4A16_ERR_LAUNCH, std::string("kernel launch failed: ") + hipGetErrorString(e));
    return W4A16_OK;
}

}  // namespace

extern "C" {

int w4a16_kv_fork(const w4a16_kv_cache* from, const w4a16_kv_cache* to, const int64_t* source, const int64_t* lengths,
                  void* stream) {
    int rc = w4a16_internal::check_kv_cache(from);
    if (rc != W4A16_OK || (rc = w4a16_internal::check_kv_cache(to)) != W4A16_OK) return rc;
    if (from->kv_heads != to->kv_heads || from->head_dim != to->head_dim || from->block != to->block ||
        from->code_type != to->code_type)
        return kv_fail(W4A16_ERR_SHAPE, "the two caches must have the same KV heads, head_dim, block and codes");
    if (to->batch == 0 || from->batch == 0) return W4A16_OK;
    if (source == nullptr || lengths == nullptr) return kv_fail(W4A16_ERR_NULL, "source and lengths must be non-NULL");
    MoveArgs a = args_of(*from, *to, source, lengths);
    a.chunk = 256 * kForkUnits / a.units;
    a.chunks = (int)((a.slots + a.chunk - 1) / a.chunk);
    const __int128 grid = (__int128)2 * a.chunks * a.kv_heads * a.batch;
    if (!w4a16_internal::launch_fits(grid, 256)) return kv_fail(W4A16_ERR_TOO_LARGE, "too many sequences for one launch");
    if ((rc = w4a16_internal::check_written(*to)) != W4A16_OK) return rc;
    if ((rc = w4a16_internal::check_apart(*from, *to)) != W4A16_OK) return rc;
    const dim3 g((unsigned)grid), t(256);
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (is_far(*to))
        hipLaunchKernelGGL((fork_kernel<true>), g, t, 0, st, a);
    else
        hipLaunchKernelGGL((fork_kernel<false>), g, t, 0, st, a);
    return finish();
}

int w4a16_kv_reorder(const w4a16_kv_cache* cache, const int64_t* source, const int64_t* lengths, void* stream) {
    int rc = w4a16_internal::check_kv_cache(cache);
    if (rc != W4A16_OK) return rc;
    if (cache->batch == 0) return W4A16_OK;
    if (source == nullptr || lengths == nullptr) return kv_fail(W4A16_ERR_NULL, "source and lengths must be non-NULL");
    MoveArgs a = args_of(*cache, *cache, source, lengths);
    const int64_t slot = cache->batch * a.units;   // units of a slot of all sequences
    const int threads = slot <= 256 * 16 ? 256 : 1024;
    if (slot > 1024 * 16)
        return kv_fail(W4A16_ERR_TOO_LARGE, "a cache that is reordered may have at most 262144 / head_dim sequences");
    const int units = slot <= 256 * 4 ? 4 : 16;
    a.chunk = (int)(threads * units / slot);
    a.chunks = (int)((a.slots + a.chunk - 1) / a.chunk);
    const __int128 grid = (__int128)2 * a.chunks * a.kv_heads;
    if (!w4a16_internal::launch_fits(grid, threads)) return kv_fail(W4A16_ERR_TOO_LARGE, "too many slots for one launch");
    if ((rc = w4a16_internal::check_written(*cache)) != W4A16_OK) return rc;
    const dim3 g((unsigned)grid), t((unsigned)threads);
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (threads == 1024)
        hipLaunchKernelGGL((reorder_kernel<1024, 16, true>), g, t, 0, st, a);
    else if (units == 16)
        hipLaunchKernelGGL((reorder_kernel<256, 16, true>), g, t, 0, st, a);
    else if (is_far(*cache))
        hipLaunchKernelGGL((reorder_kernel<256, 4, true>), g, t, 0, st, a);
    else
        hipLaunchKernelGGL((reorder_kernel<256, 4, false>), g, t, 0, st, a);
    return finish();
}

}  // extern "C"
