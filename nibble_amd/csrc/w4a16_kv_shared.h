// Kernels of attention behind shared prefixes (include/w4a16_kv.h) and their
// launches for one head_dim. The attending ones are those of w4a16_kv_attn.h.
//
// Mathematics. The softmax over a prefix and a sequence's own slots is that over
// the two apart, joined by their states: with R, l, o of each share s,
//     out = sum_s o_s 2^(R_s - R) / sum_s l_s 2^(R_s - R).
// So the rows of all sequences behind one prefix attend it together, as the rows
// of one long sequence would, and a key or value of the prefix is read once for
// all of them.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "w4a16_kv_attn.h"

namespace w4a16 {

// ---------------------------------------------------------------------------
// The shares of an output row joined, by W wavefronts (a workgroup of 256
// threads joins 4 / W rows). Lane s holds share s's state (at most 64): those of
// the prefix first, then the sequence's own. `unit` slots a chunk or tile of the
// launches before, `own_rows` rows a workgroup of the own slots' launch: they give
// the shares that were written.
//
// Bound: latency, of the lengths' chain of loads and one round of shares (2048 rows
// of 11 shares of 128 dims, 11.5 MB: 5.7 us; 512 rows of 13 of 64 dims 4.3).
// ---------------------------------------------------------------------------
template <int D, int TYPE, int W>
__global__ void __launch_bounds__(256) join_kernel(const AttnArgs prefix, const AttnArgs own, int prefix_unit,
                                                   int own_unit, int own_rows, int64_t rows) {
    constexpr int E = D / 64;   // dims a lane
    constexpr int F = W == 1 ? 12 : 4;   // shares of a wavefront in flight
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

// ---------------------------------------------------------------------------
// Prefix and own slots in one launch, both in the decode form, so that the short
// side costs no launch and fills what the long one leaves.
//
// Bound: the prefixes' bytes (4 of 30001 slots, 4 KV heads of 128, 42 rows each: 35
// us, 3.5 TB/s; in the prompt form, which decodes through LDS, 59 with its join).
// ---------------------------------------------------------------------------
template <int D, int NTP, int NTO, int CODES, int TYPE>
__global__ void __launch_bounds__(64 * kDecodeWaves, decode_workgroups(D, NTP))
pair_kernel(const AttnArgs prefix, const OwnArgs own) {
    __shared__ union {
        DecodeLds<D, NTP> prefix;
        DecodeLds<D, NTO> own;
    } lds;
    if ((int)blockIdx.x < own.prefix_blocks)
        decode_body<D, NTP, CODES, TYPE, Prefix>(prefix, blockIdx.x, lds.prefix);
    else
        decode_body<D, NTO, CODES, TYPE, Own>(own.args, (int)blockIdx.x - own.prefix_blocks, lds.own);
}

// How one side (a prefix, or the sequences' own slots) is launched.
struct SidePlan {
    bool prompt;
    int waves;          // W of the prompt form
    int column_tiles;   // NT of the decode form
    int rows_per;
    int64_t row_tiles;
    int unit;           // slots of a chunk or tile
    int splits, least;
    int threads;
};

// Wavefronts of the prompt form on a prefix alone, and on own slots where these give many
// workgroups (which then have one share, so that Last is their mode).
constexpr int wide_waves(int dim) { return dim <= 128 ? 8 : 4; }

struct SharedPlan {
    SidePlan prefix, own;
    bool last;          // the own slots' launch joins the prefix's shares, else a launch of its own does
    int pitch;          // shares of a row that are written
};

struct SharedCall {
    SharedPlan plan;
    AttnArgs prefix, own;
    int64_t prefix_grid, own_grid, rows;
    hipStream_t stream;
};

template <int D, int NTP, int NTO, int CODES, int TYPE>
void launch_pair(const SharedCall& c) {
    const dim3 grid((unsigned)(c.prefix_grid + c.own_grid)), threads(64 * kDecodeWaves);
    hipLaunchKernelGGL((pair_kernel<D, NTP, NTO, CODES, TYPE>), grid, threads, 0, c.stream, c.prefix,
                       (OwnArgs{c.own, (int)c.prefix_grid}));
}

template <int D, int NTO, int CODES, int TYPE>
void launch_beside(const SharedCall& c) {   // own slots in the decode form
    const SidePlan& p = c.plan.prefix;
    if (p.prompt) {
        const dim3 grid((unsigned)(c.prefix_grid + c.own_grid)), threads(64 * kDecodeWaves);
        hipLaunchKernelGGL((prompt_kernel<D, 4, 1, CODES, TYPE, Prefix, NTO, OwnArgs>), grid, threads, 0, c.stream,
                           c.prefix, (OwnArgs{c.own, (int)c.prefix_grid}));
    } else if (p.column_tiles == 3) {
        if constexpr (D == 128) launch_pair<D, 3, NTO, CODES, TYPE>(c);
    } else if (p.column_tiles == 2) {
        launch_pair<D, 2, NTO, CODES, TYPE>(c);
    } else {
        launch_pair<D, NTO == 2 ? 2 : 1, NTO, CODES, TYPE>(c);
    }
}

template <int D, int W, int CODES, int TYPE, Mode MODE>
void launch_prompt(const AttnArgs& a, int64_t grid, hipStream_t st) {
    hipLaunchKernelGGL((prompt_kernel<D, W, 1, CODES, TYPE, MODE>), dim3((unsigned)grid), dim3(64 * W), 0, st, a);
}

template <int D, int CODES, int TYPE>
void launch_codes(const SharedCall& c) {
    if (!c.plan.own.prompt) {
        if (c.plan.own.column_tiles == 1)
            launch_beside<D, 1, CODES, TYPE>(c);
        else
            launch_beside<D, 2, CODES, TYPE>(c);
    } else {
        constexpr int WIDE = wide_waves(D);
        launch_prompt<D, WIDE, CODES, TYPE, Prefix>(c.prefix, c.prefix_grid, c.stream);
        if (c.plan.last) {
            if (c.plan.own.waves == WIDE)
                launch_prompt<D, WIDE, CODES, TYPE, Last>(c.own, c.own_grid, c.stream);
            else
                launch_prompt<D, 4, CODES, TYPE, Last>(c.own, c.own_grid, c.stream);
            return;
        }
        launch_prompt<D, 4, CODES, TYPE, Own>(c.own, c.own_grid, c.stream);
    }
    const dim3 threads(256);
    // a wavefront a row where there are many rows of few shares (2048 rows of 11: 37
    // against 40 us with the launch before; 512 rows of 13: 12.7 against 11.8)
    if (c.rows <= 1024 ? c.plan.pitch > 4 : c.plan.pitch > 16)
        hipLaunchKernelGGL((join_kernel<D, TYPE, 4>), dim3((unsigned)c.rows), threads, 0, c.stream, c.prefix, c.own,
                           c.plan.prefix.unit, c.plan.own.unit, c.plan.own.rows_per, c.rows);
    else
        hipLaunchKernelGGL((join_kernel<D, TYPE, 1>), dim3((unsigned)((c.rows + 3) / 4)), threads, 0, c.stream,
                           c.prefix, c.own, c.plan.prefix.unit, c.plan.own.unit, c.plan.own.rows_per, c.rows);
}

template <int D>
void launch_shared(const SharedCall& c, int code_type, int type) {
    if (code_type == W4A16_KV_INT8 && type == W4A16_FP16)
        launch_codes<D, W4A16_KV_INT8, W4A16_FP16>(c);
    else if (code_type == W4A16_KV_INT8)
        launch_codes<D, W4A16_KV_INT8, W4A16_BF16>(c);
    else if (type == W4A16_FP16)
        launch_codes<D, W4A16_KV_FP8, W4A16_FP16>(c);
    else
        launch_codes<D, W4A16_KV_FP8, W4A16_BF16>(c);
}

// a source file each, as they take a minute to compile
extern template void launch_shared<64>(const SharedCall&, int, int);
extern template void launch_shared<128>(const SharedCall&, int, int);
extern template void launch_shared<256>(const SharedCall&, int, int);

}  // namespace w4a16
