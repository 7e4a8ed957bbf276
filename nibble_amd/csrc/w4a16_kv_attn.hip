// Attention over the 8-bit key/value cache (include/w4a16_kv.h).
//
// Mathematics. The query rows of one KV head, r = t group + g (token t, query
// head g of the head's group), attend together, so that a key or value is
// read once for all of them. With e_k, e_v the exponents of the scales of slot
// j's blocks, the score in powers of two is
//     s_j = (q . code_k,j) 2^e_k scale log2(e),
// and the value's scale joins the softmax instead of the product:
//     w_j = s_j + e_v,   R ~ max_j w_j - 7,   P_j = 2^(w_j - R),
//     o = sum_j P_j code_v,j / sum_j 2^-e_v P_j.
// Both products run on the matrix cores with fp16 operands. Codes are exact in
// fp16, fp16 queries too; bf16 rows are moved into fp16's range by a power of
// two per row, exact for values down to 2^-31 of the row's largest and off by
// 2^-39 of it below. P is rounded to fp16, by 2^-11 of itself for weights down
// to 2^-21 of the row's largest P, by 2^-32 of that below (kBelow). Scores, R,
// both sums and the outputs are fp32.
//
// S^T = K Q^T and O^T = V^T P^T: with keys in the rows of the first product a
// lane receives weights of consecutive keys of its own query column, which are
// the second product's right operand as they stand, if V^T's keys are taken in
// the same order. Neither P nor, in the decode form, K and V pass through LDS.
#include <hip/hip_runtime.h>

#include <cstdint>
#include <string>

#include "w4a16_hip.h"
#include "w4a16_kv_device.h"
#include "w4a16_kv_host.h"

namespace w4a16 {

typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr float kLog2e = 1.4426950408889634f;

struct AttnArgs {
    const uint16_t* q;
    uint16_t* out;
    const uint8_t *k_codes, *v_codes;
    const float *k_scales, *v_scales;
    const int64_t *start, *counts;
    float2* states;   // [batch tokens heads][splits] {R, l} and
    float* partial;   // [batch tokens heads][splits][dim], with splits > 1
    int64_t qb, qt, qh;
    int64_t kb, kh, vb, vh, ksb, ksh, vsb, vsh;
    int64_t slots;
    float scale;
    int tokens, heads, kv_heads, group, block_log, splits, least, row_tiles;
    bool vec;
    bool early;   // shares request their first chunk before `start` has arrived
};

// What a workgroup's rows see: rows row0 .. of sequence b.
struct Seen {
    int64_t start;
    int count;   // tokens that are no padding
};

__device__ __forceinline__ Seen seen_of(const AttnArgs& a, int b) {
    Seen s;
    s.start = min(a.start[b], a.slots);   // past the slots: no row is inside
    s.count = a.tokens;
    if (a.counts != nullptr) s.count = (int)min(max(a.counts[b], (int64_t)0), (int64_t)a.tokens);
    return s;
}

// Slots that the rows row0 .. row0 + n - 1 see together: 0 .. end - 1.
__device__ __forceinline__ int seen_end(const AttnArgs& a, const Seen& s, int row0, int n) {
    const int last_row = min(row0 + n, a.tokens * a.group) - 1;
    const int t = min(last_row / a.group, s.count - 1);
    if (t < row0 / a.group) return 0;
    const int64_t p = min(s.start + t, a.slots - 1);
    return p < 0 ? 0 : (int)p + 1;
}

// The shares that a workgroup's `parts` chunks or tiles are divided into:
// `splits` of them at most, none of fewer than `least`, one up to three times
// that. One share writes the outputs itself; with more each writes its state,
// and merge_kernel joins them.
struct Shares {
    int size, count;
};
__host__ __device__ __forceinline__ Shares shares_of(int parts, int splits, int least) {
    const int even = (parts + splits - 1) / splits;
    const int size = parts <= 3 * least ? (parts > 0 ? parts : 1) : even > least ? even : least;
    return {size, (parts + size - 1) / size};
}

// A query row's 16-bit values -> fp16, with the power of two that was divided
// out (bf16 only). The row's values are spread over the lanes that `rowmax`
// joins.
template <int TYPE, int N, typename F>
__device__ __forceinline__ float query_to_f16(u32x4 (&q)[N], F rowmax) {
    if constexpr (TYPE == W4A16_FP16) {
        return 1.0f;
    } else {
        float amax = 0.0f;
        float x[N][8];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            widen8<TYPE>(q[i], x[i]);
#pragma unroll
            for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fabsf(x[i][e]));
        }
        amax = rowmax(amax);
        // the largest magnitude to 2^14 .. 2^15; infinities and zeros keep a shift that a float holds
        int shift = 14 - ((int)(__builtin_bit_cast(uint32_t, amax) >> 23) - 127);
        shift = min(max(shift, -120), 120);
        const float m = exp2_int(shift);
#pragma unroll
        for (int i = 0; i < N; ++i) {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[i][e] *= m;
            q[i] = narrow8<W4A16_FP16>(x[i]);
        }
        return exp2_int(-shift);
    }
}

// 8 codes (two biased words) as a matrix operand.
template <int CODES>
__device__ __forceinline__ f16x8 decode8(uint32_t a, uint32_t b) {
    a = kv_bias<CODES>(a);
    b = kv_bias<CODES>(b);
    const u32x4 v = {as_u32(decode2_f16<CODES, false>(a)), as_u32(decode2_f16<CODES, true>(a)),
                     as_u32(decode2_f16<CODES, false>(b)), as_u32(decode2_f16<CODES, true>(b))};
    return __builtin_bit_cast(f16x8, v);
}

// Words x[0..7] of 8 slots, 4 dims each -> for each dim the 8 slots' values as a
// matrix operand. Byte pairs of neighbouring keys come together by v_perm.
template <int CODES>
__device__ __forceinline__ void transpose8(const uint32_t (&x)[8], f16x8 (&out)[4]) {
    u32x4 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t lo = kv_bias<CODES>(perm(x[2 * i + 1], x[2 * i], 0x05010400u));   // dims 0, 1
        const uint32_t hi = kv_bias<CODES>(perm(x[2 * i + 1], x[2 * i], 0x07030602u));   // dims 2, 3
        v[0][i] = as_u32(decode2_f16<CODES, false>(lo));
        v[1][i] = as_u32(decode2_f16<CODES, true>(lo));
        v[2][i] = as_u32(decode2_f16<CODES, false>(hi));
        v[3][i] = as_u32(decode2_f16<CODES, true>(hi));
    }
#pragma unroll
    for (int d = 0; d < 4; ++d) out[d] = __builtin_bit_cast(f16x8, v[d]);
}

// 4 consecutive outputs of a row.
template <int TYPE>
__device__ __forceinline__ void store4(uint16_t* p, float a, float b, float c, float d) {
    *reinterpret_cast<uint2*>(p) = make_uint2(narrow16<TYPE>(a) | (narrow16<TYPE>(b) << 16),
                                              narrow16<TYPE>(c) | (narrow16<TYPE>(d) << 16));
}

// The larger of two values without the quieting of signalling NaN that fmaxf
// brings (an instruction for each operand that a matrix product left).
__device__ __forceinline__ float larger(float a, float b) {
    return __builtin_amdgcn_fmed3f(a, b, __builtin_inff());
}

// A row's reference R of the weights 2^(w - R) lies kBelow under its largest w,
// and follows that only when a weight would pass 2^kMost, so that the outputs
// are rarely rescaled. fp16 ends at 2^16 and is normal down to 2^-14: a weight
// is off by 2^-11 of itself down to 2^-21 of the row's largest, below by 2^-32
// of the largest. (With R at the largest w, weights under 2^-25 of it are lost:
// a prompt's row over 131071 slots of score 0 and one of score 17.5 whose value
// is 0 came out 0 where 0.026 was right.)
constexpr float kBelow = 7.0f, kMost = 15.0f;

// R after larger weights w <= mx came: -inf as long as there were none.
__device__ __forceinline__ float reference(float mx, float before) { return fmaxf(mx - kBelow, before); }

// ---------------------------------------------------------------------------
// Decode form: up to 16 NT query rows of a KV head, every wavefront taking
// chunks of 16 M slots.
//
// Bound: the cache's bytes with many sequences (32 of 7000 tokens, 8 KV heads of
// 128: 84.7 us, 5.5 TB/s), the latency of a chunk (about 1.5 us from request to
// output) with few. Lane (c, h) = (lane & 15, lane >> 4).
// Keys: 16 bytes of row c at 64 j + 16 h, so that the loads of a row read it
// whole; values: dim / 16 bytes at dim / 16 c of the rows that the lane's
// weights stand for (slots 32 y + 4 h + i and 32 y + 16 + 4 h + i), whole rows
// again. The next chunk's keys are requested when the present ones are
// multiplied, its values likewise. Wavefronts of a workgroup join through LDS;
// the chunks of a sequence go round the shares, which merge_kernel joins. Which
// chunk comes first does not depend on the sequence's length, so that it is
// requested before `start` has arrived.
// ---------------------------------------------------------------------------
constexpr int kDecodeWaves = 4;
// M, the 16-slot tiles of a chunk: four where they leave registers for two
// wavefronts a SIMD, as the latency of a chunk is paid once for more of them
// (one token over 8000 slots, 8 KV heads of 128, in one share: 63 us against 76
// with two); two with more rows (20 rows over 131072 slots of int8: 63 us against 73).
constexpr int chunk_tiles(int dim, int column_tiles) { return dim == 256 || column_tiles > 1 ? 2 : 4; }

template <int D, int NT, int CODES, int TYPE>
__global__ void __launch_bounds__(64 * kDecodeWaves, D * NT > 256 || D == 256 ? 1 : 2)
decode_kernel(const AttnArgs a) {
    constexpr int W = kDecodeWaves;
    constexpr int M = chunk_tiles(D, NT), C = 16 * M;
    constexpr int J = D / 64;                    // 16-byte loads of a key row's quarter; words of a value load
    constexpr int PARTS = D > 128 ? D / 128 : 1;
    constexpr int DP = D / PARTS;
    __shared__ float row_max[W][16 * NT], row_sum[W][16 * NT];
    __shared__ __align__(16) float joined[W][16][DP + 4];

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    const int c = lane & 15, h = lane >> 4;
    int item = blockIdx.x;
    const int split = item % a.splits;
    item /= a.splits;
    const int tile = item % a.row_tiles;
    item /= a.row_tiles;
    const int hk = item % a.kv_heads, b = item / a.kv_heads;
    const int rows = a.tokens * a.group, row0 = tile * 16 * NT;

    const uint8_t* kc = a.k_codes + b * a.kb + hk * a.kh;
    const uint8_t* vc = a.v_codes + b * a.vb + hk * a.vh;
    const float* ks = a.k_scales + b * a.ksb + hk * a.ksh;
    const float* vs = a.v_scales + b * a.vsb + hk * a.vsh;
    u32x4 kr[M][J];
    uint32_t vr[M][4][J];   // rows 16 y + 4 h + i of the chunk
    float k_scale[M], v_scale[M];
    auto load_keys = [&](int chunk, int limit) {
#pragma unroll
        for (int m = 0; m < M; ++m) {
            const uint8_t* row = kc + (int64_t)min(C * chunk + 16 * m + c, limit) * D + 16 * h;
#pragma unroll
            for (int j = 0; j < J; ++j) kr[m][j] = *reinterpret_cast<const u32x4*>(row + 64 * j);
            const int at = min(C * chunk + 16 * m, limit) >> a.block_log;
            k_scale[m] = ks[at];
            v_scale[m] = vs[at];
        }
    };
    auto load_values = [&](int chunk, int limit) {
#pragma unroll
        for (int y = 0; y < M; ++y)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint8_t* row = vc + (int64_t)min(C * chunk + 16 * y + 4 * h + i, limit) * D + (D / 16) * c;
                if constexpr (J == 1) {
                    vr[y][i][0] = *reinterpret_cast<const uint32_t*>(row);
                } else if constexpr (J == 2) {
                    const uint2 v = *reinterpret_cast<const uint2*>(row);
                    vr[y][i][0] = v.x;
                    vr[y][i][1] = v.y;
                } else {
                    const u32x4 v = *reinterpret_cast<const u32x4*>(row);
#pragma unroll
                    for (int w = 0; w < 4; ++w) vr[y][i][w] = v[w];
                }
            }
    };
    // (where the cache is large the other shares, which may turn out to have no
    // slots, read the first rows here and their own below: registers that only
    // one side of a branch defines have been miscompiled)
    int chunk = split * W + wave;
    const bool early = split == 0 || a.early;
    load_keys(early ? chunk : 0, (int)a.slots - 1);
    load_values(early ? chunk : 0, (int)a.slots - 1);

    u32x4 qr[NT][2 * J];
    float row_scale[NT];
    int last[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int r = min(row0 + 16 * n + c, rows - 1);
        const int t = r / a.group, g = r - t * a.group;
        const uint16_t* q = a.q + b * a.qb + t * a.qt + (hk * a.group + g) * a.qh;
#pragma unroll
        for (int j = 0; j < J; ++j) {
            qr[n][2 * j] = load8(q + 64 * j + 16 * h, a.vec);
            qr[n][2 * j + 1] = load8(q + 64 * j + 16 * h + 8, a.vec);
        }
    }
    const Seen seen = seen_of(a, b);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int t = min(row0 + 16 * n + c, rows - 1) / a.group;
        const int64_t p = seen.start + t;
        last[n] = t < seen.count && p >= 0 && p < a.slots ? (int)p : -1;
    }
    const int end = seen_end(a, seen, row0, 16 * NT);
    const int last_slot = max(end - 1, 0);
    const int chunks = (end + C - 1) / C;
    const Shares shares = shares_of(chunks, a.splits, a.least);
    if (split > 0 && split >= shares.count) return;
    if (!early) {
        load_keys(chunk, last_slot);
        load_values(chunk, last_slot);
    }
    const int step = W * max(shares.count, 1);
#pragma unroll
    for (int n = 0; n < NT; ++n)
        row_scale[n] = a.scale * kLog2e * query_to_f16<TYPE>(qr[n], row_pair_max);

    float run_max[NT], run_sum[NT];
    f32x4 acc[NT][D / 16];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        run_max[n] = -__builtin_inff();
        run_sum[n] = 0.0f;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) acc[n][i] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
    }
    while (chunk < chunks) {
        const int slot0 = C * chunk;
        f32x4 st[NT][M];
        float ksc[M], vex[M], vinv[M];
#pragma unroll
        for (int m = 0; m < M; ++m) {
            ksc[m] = k_scale[m];
            // a tile behind the last slot may have any scale: its weights are 0, but
            // their factor has to be a number
            const int e = min(max(exponent_of(v_scale[m]), -100), 100);
            vex[m] = (float)e;
            vinv[m] = exp2_int(-e);
#pragma unroll
            for (int n = 0; n < NT; ++n) st[n][m] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int j = 0; j < J; ++j)
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const f16x8 key = decode8<CODES>(kr[m][j][2 * x], kr[m][j][2 * x + 1]);
#pragma unroll
                    for (int n = 0; n < NT; ++n)
                        st[n][m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                            key, __builtin_bit_cast(f16x8, qr[n][2 * j + x]), st[n][m], 0, 0, 0);
                }
        }
        const int next = chunk + step;
        if (next < chunks) load_keys(next, last_slot);
        f16x8 weights[NT][M / 2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            float mx = -__builtin_inff();
#pragma unroll
            for (int m = 0; m < M; ++m)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float w = __builtin_fmaf(st[n][m][e], row_scale[n] * ksc[m], vex[m]);
                    if (slot0 + 16 * m + 4 * h + e > last[n]) w = -__builtin_inff();
                    st[n][m][e] = w;
                    mx = larger(mx, w);
                }
            mx = row_pair_max(mx);
            if (__any(mx - run_max[n] > kMost)) {
                mx = reference(mx, run_max[n]);
                const float rescale = mx == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(run_max[n] - mx);
                run_max[n] = mx;
                run_sum[n] *= rescale;
#pragma unroll
                for (int i = 0; i < D / 16; ++i) acc[n][i] *= rescale;
            }
            const float base = run_max[n] == -__builtin_inff() ? 0.0f : run_max[n];   // no slot of the row seen yet
#pragma unroll
            for (int y = 0; y < M / 2; ++y) {
                u32x4 packed;
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const int m = 2 * y + x;
                    float p[4], sum = 0.0f;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        p[e] = __builtin_amdgcn_exp2f(st[n][m][e] - base);
                        sum += p[e];
                    }
                    run_sum[n] = __builtin_fmaf(sum, vinv[m], run_sum[n]);
                    packed[2 * x] = as_u32((f16x2){(f16)p[0], (f16)p[1]});
                    packed[2 * x + 1] = as_u32((f16x2){(f16)p[2], (f16)p[3]});
                }
                weights[n][y] = __builtin_bit_cast(f16x8, packed);
            }
        }
        if (slot0 + C > end) {   // rows behind the last slot may hold anything, NaN codes too
#pragma unroll
            for (int y = 0; y < M; ++y)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (slot0 + 16 * y + 4 * h + i >= end)
#pragma unroll
                        for (int j = 0; j < J; ++j) vr[y][i][j] = 0;
        }
#pragma unroll
        for (int y = 0; y < M / 2; ++y)
#pragma unroll
            for (int j = 0; j < J; ++j) {
                uint32_t words[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) words[i] = vr[2 * y + (i >> 2)][i & 3][j];
                f16x8 value[4];
                transpose8<CODES>(words, value);
#pragma unroll
                for (int d = 0; d < 4; ++d)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
                        acc[n][4 * j + d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(value[d], weights[n][y],
                                                                                   acc[n][4 * j + d], 0, 0, 0);
            }
        if (next >= chunks) break;
        chunk = next;
        load_values(chunk, last_slot);
    }

    // the wavefronts' states joined: lane (c, h) holds row c's dims D / 16 (4 h + i) + j in acc[][j][i]
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        run_sum[n] = row_pair_sum(run_sum[n]);
        if (h == 0) {
            row_max[wave][16 * n + c] = run_max[n];
            row_sum[wave][16 * n + c] = run_sum[n];
        }
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        float top = row_max[0][16 * n + c];
#pragma unroll
        for (int w = 1; w < W; ++w) top = fmaxf(top, row_max[w][16 * n + c]);
        const float own = run_max[n] == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(run_max[n] - top);
#pragma unroll
        for (int part = 0; part < PARTS; ++part) {
            if (n + part > 0) __syncthreads();   // the previous values are read
#pragma unroll
            for (int i = 0; i < 4 / PARTS; ++i)
#pragma unroll
                for (int j = 0; j < D / 16; j += 4) {
                    const int e = part * (4 / PARTS) + i;
                    *reinterpret_cast<f32x4*>(&joined[wave][c][(D / 16) * ((4 / PARTS) * h + i) + j]) =
                        (f32x4){acc[n][j][e], acc[n][j + 1][e], acc[n][j + 2][e], acc[n][j + 3][e]} * own;
                }
            __syncthreads();
            for (int x = threadIdx.x; x < 16 * DP / 4; x += 64 * W) {
                const int row = x / (DP / 4), col = 4 * (x - row * (DP / 4));
                const int r = row0 + 16 * n + row;
                if (r >= rows) continue;
                f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
                float t0 = -__builtin_inff(), l = 0.0f;
#pragma unroll
                for (int w = 0; w < W; ++w) t0 = fmaxf(t0, row_max[w][16 * n + row]);
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    o += *reinterpret_cast<const f32x4*>(&joined[w][row][col]);
                    const float m = row_max[w][16 * n + row];
                    l += m == -__builtin_inff() ? 0.0f : row_sum[w][16 * n + row] * __builtin_amdgcn_exp2f(m - t0);
                }
                // the column in `joined` -> the head's dim (256 dims come in two parts)
                const int q = col / (D / 16), dim = PARTS == 1 ? col
                    : (D / 16) * (4 * (q / (4 / PARTS)) + part * (4 / PARTS) + q % (4 / PARTS)) + col % (D / 16);
                const int t = r / a.group, g = r - t * a.group;
                const int64_t at = ((int64_t)b * a.tokens + t) * a.heads + hk * a.group + g;
                if (shares.count > 1) {
                    const int64_t sp = at * a.splits + split;
                    *reinterpret_cast<f32x4*>(a.partial + sp * D + dim) = o;
                    if (col == 0 && part == 0) a.states[sp] = make_float2(t0, l);
                    continue;
                }
                const int64_t p = seen.start + t;
                float inv = 1.0f / l;
                if (t >= seen.count) {
                    o = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
                    inv = 0.0f;
                } else if (p < 0 || p >= a.slots) {
                    inv = __builtin_nanf("");
                }
                store4<TYPE>(a.out + at * D + dim, o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
            }
        }
    }
}

// The shares of an output row joined by a workgroup: out = sum_s acc_s 2^(R_s
// - R) / sum_s l_s 2^(R_s - R). Lane s holds share s's state (at most 64
// shares); wavefront w takes the shares w, w + 4, .., four in flight.
// `rows_per` rows make a workgroup of the launch before, `unit` slots a chunk
// or tile of it: they give the shares that were written.
template <int D, int TYPE>
__global__ void __launch_bounds__(256) merge_kernel(const AttnArgs a, int rows_per, int unit) {
    constexpr int E = D / 64;   // dims a lane
    constexpr int F = 4;        // shares of a wavefront in flight
    __shared__ float parts[4][D];
    const int64_t row = blockIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const float* part = a.partial + row * a.splits * D + lane * E;
    float v[F][E];
    auto load = [&](int s0) {
#pragma unroll
        for (int x = 0; x < F; ++x)
#pragma unroll
            for (int e = 0; e < E; ++e) v[x][e] = part[(int64_t)min(s0 + 4 * x, a.splits - 1) * D + e];
    };
    // requested before `start` tells which of them were written
    load(wave);
    float2 state = a.states[row * a.splits + min(lane, a.splits - 1)];
    const int64_t bt = row / a.heads;
    const int head = (int)(row - bt * a.heads);
    const int b = (int)(bt / a.tokens), t = (int)(bt - (int64_t)b * a.tokens);
    const Seen seen = seen_of(a, b);
    const int r = t * a.group + head % a.group;
    const int end = seen_end(a, seen, r - r % rows_per, rows_per);
    const int count = shares_of((end + unit - 1) / unit, a.splits, a.least).count;
    if (count < 2) return;   // the one share has written the row
    const int64_t p = seen.start + t;
    const bool inside = t < seen.count && p >= 0 && p < a.slots;   // else nothing was written
    if (!inside || lane >= count) state = make_float2(-__builtin_inff(), 0.0f);
    float o[E] = {};
    const float top = wave_max(state.x);
    const float f = state.x == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(state.x - top);
    if (inside) {
        for (int s0 = wave; s0 < count; s0 += 4 * F) {
#pragma unroll
            for (int x = 0; x < F; ++x) {
                const int s = s0 + 4 * x;
                const float fs = __builtin_bit_cast(
                    float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, f), min(s, count - 1)));
#pragma unroll
                for (int e = 0; e < E; ++e) o[e] = s < count ? __builtin_fmaf(v[x][e], fs, o[e]) : o[e];
            }
            if (s0 + 4 * F < count) load(s0 + 4 * F);
        }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) parts[wave][lane * E + e] = o[e];
    __syncthreads();
    if (wave != 0) return;
    const float inv = t >= seen.count ? 0.0f : inside ? 1.0f / wave_sum(state.y * f) : __builtin_nanf("");
    uint16_t* out = a.out + row * D + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e)
        out[e] = (uint16_t)narrow16<TYPE>(((parts[0][lane * E + e] + parts[1][lane * E + e]) +
                                           (parts[2][lane * E + e] + parts[3][lane * E + e])) * inv);
}

// The prompt form takes w - R in one step, (q . code_k) mul + (e_v - R), where R
// came from w's rounded to fp32. From this size of R on their roundings together
// reach a unit of the exponent and more, up to weights that fp16 does not hold or
// that are all 0: a wavefront that met such an R attends its rows once more by
// attend_row, which forms w first and takes R off after, as the decode form does.
constexpr float kLarge = 0x1p22f;

// Row r of a KV head over the slots from `lo` to `hi`, by one wavefront and in
// fp32 throughout: a lane a slot for the scores, D / 64 dims a lane for the
// outputs. `split` is the share, -1 where there is one. Right for scores of any
// size, and slow: 4096 tokens of 32/8 heads of 128 in 19 ms.
template <int D, int CODES, int TYPE>
__device__ __forceinline__ void attend_row(const AttnArgs& a, const Seen& seen, int b, int hk, int r, int64_t lo,
                                           int64_t hi, int split) {
    constexpr int E = D / 64;
    const int lane = threadIdx.x & 63;
    const int t = r / a.group, g = r - t * a.group;
    const int64_t p = seen.start + t;
    const bool inside = t < seen.count && p >= 0 && p < a.slots;
    hi = inside ? min(hi, p + 1) : lo;
    const uint16_t* q = a.q + b * a.qb + t * a.qt + (hk * a.group + g) * a.qh;
    const uint8_t* kc = a.k_codes + b * a.kb + hk * a.kh;
    const uint8_t* vc = a.v_codes + b * a.vb + hk * a.vh + lane * E;
    const float* ks = a.k_scales + b * a.ksb + hk * a.ksh;
    const float* vs = a.v_scales + b * a.vsb + hk * a.vsh;
    // bf16 queries may be of any size: a power of two brings the largest to 2^14 .. 2^15
    float amax = 0.0f;
    for (int i = 0; i < E; ++i) amax = fmaxf(amax, fabsf(widen16<TYPE>(q[lane * E + i])));
    const int shift = min(max(14 - exponent_of(wave_max(amax)), -120), 120);
    const float m = exp2_int(shift), row_scale = a.scale * kLog2e * exp2_int(-shift);
    float top = -__builtin_inff(), sum = 0.0f, o[E] = {};
    for (int64_t slot0 = lo; slot0 < hi; slot0 += 64) {
        const int64_t slot = min(slot0 + lane, hi - 1);
        float dot = 0.0f;
        for (int d = 0; d < D; d += 4) {
            const uint32_t word = *reinterpret_cast<const uint32_t*>(kc + slot * D + d);
            const f32x2 x = decode2_f32<CODES, false>(word), y = decode2_f32<CODES, true>(word);
            dot = __builtin_fmaf(widen16<TYPE>(q[d]) * m, x.x, dot);
            dot = __builtin_fmaf(widen16<TYPE>(q[d + 1]) * m, x.y, dot);
            dot = __builtin_fmaf(widen16<TYPE>(q[d + 2]) * m, y.x, dot);
            dot = __builtin_fmaf(widen16<TYPE>(q[d + 3]) * m, y.y, dot);
        }
        const int e = exponent_of(vs[slot >> a.block_log]);
        float w = __builtin_fmaf(dot, row_scale * ks[slot >> a.block_log], (float)e);
        if (slot0 + lane >= hi) w = -__builtin_inff();
        const float mx = fmaxf(wave_max(w), top);
        const float rescale = top == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(top - mx);
        top = mx;
        const float weight = __builtin_amdgcn_exp2f(w - top);
        sum = __builtin_fmaf(sum, rescale, weight * exp2_int(-e));
        for (int i = 0; i < E; ++i) o[i] *= rescale;
        const int n = (int)min(hi - slot0, (int64_t)64);
        for (int j = 0; j < n; ++j) {
            const float x = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, weight), j));
            uint32_t word = 0;
            for (int i = 0; i < E; ++i) word |= (uint32_t)vc[(slot0 + j) * D + i] << (8 * i);
            const f32x2 lower = decode2_f32<CODES, false>(word), upper = decode2_f32<CODES, true>(word);
            const float value[4] = {lower.x, lower.y, upper.x, upper.y};
            for (int i = 0; i < E; ++i) o[i] = __builtin_fmaf(x, value[i], o[i]);
        }
    }
    sum = wave_sum(sum);
    const int64_t at = ((int64_t)b * a.tokens + t) * a.heads + hk * a.group + g;
    if (split >= 0) {
        const int64_t sp = at * a.splits + split;
        for (int i = 0; i < E; ++i) a.partial[sp * D + lane * E + i] = o[i];
        if (lane == 0) a.states[sp] = make_float2(top, sum);
        return;
    }
    const float inv = t >= seen.count ? 0.0f : inside ? 1.0f / sum : __builtin_nanf("");
    for (int i = 0; i < E; ++i) a.out[at * D + lane * E + i] = (uint16_t)narrow16<TYPE>(o[i] * inv);
}

// ---------------------------------------------------------------------------
// Prompt form: 32 W query rows of a KV head a workgroup, 32 a wavefront.
//
// Bound: the matrix cores and the softmax's vector instructions together (4 dim
// flops a pair of row and slot; 4096 tokens of 32/8 heads of 128: 151 us, 912
// TFLOP/s, two thirds of what an 8192^3 product reaches; the counters show the
// matrix cores busy 45% of the time, the vector unit 54%, LDS 31%: two
// wavefronts a SIMD, which the registers allow, do not cover each other's
// waits). Tiles of 64 slots (32 with head_dim 256): their codes are requested
// into registers a tile and a half ahead, decoded to fp16 once for the
// workgroup's rows and kept in LDS, keys row by row, values transposed with
// their slots in the order of the score registers.
// v_mfma_f32_32x32x16_f16: lane (n, h) = (lane & 31, lane >> 5) receives the
// scores of row n for slots 8 (i >> 2) + 4 h + (i & 3) of each 32.
// ---------------------------------------------------------------------------
__device__ __forceinline__ float half_pair_max(float v) {   // over lanes l and l ^ 32
    const auto x = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v),
                                                    false, false);
    return fmaxf(__builtin_bit_cast(float, (uint32_t)x[0]), __builtin_bit_cast(float, (uint32_t)x[1]));
}
__device__ __forceinline__ float half_pair_sum(float v) {
    const auto x = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v),
                                                    false, false);
    return __builtin_bit_cast(float, (uint32_t)x[0]) + __builtin_bit_cast(float, (uint32_t)x[1]);
}

// head_dim 256 keeps its outputs and queries in 512 registers, one wavefront a SIMD
template <int D, int W, int KS, int CODES, int TYPE>
__global__ void __launch_bounds__(64 * W * KS, D == 256 ? 1 : 2)
prompt_kernel(const AttnArgs a) {
    constexpr int KT = D == 256 ? 32 : 64;   // slots of a tile
    constexpr int KN = KT / 32;
    constexpr int KROW = D + 8;              // fp16 values of a key row in LDS
    constexpr int VROW = KT + 8;             // of a value dim's row
    constexpr int KU = KT * D / 16;          // 16-byte units of a tile's keys
    constexpr int KL = KU > 64 * W ? KU / (64 * W) : 1;   // of a thread
    constexpr int KW = KU < 64 * W ? KU / 64 : W;         // wavefronts that load keys: the first ones
    constexpr int VW = KT * D / 32 / 64;                  // and values: the last ones
    constexpr int KSIZE = KT * KROW, VSIZE = D * VROW;
    __shared__ __align__(16) f16 staged[KS][2 * (KSIZE + VSIZE)];

    // KS groups of W wavefronts attend the same rows, each every KS-th tile
    const int group = KS == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / (64 * W));
    const int tid = KS == 1 ? (int)threadIdx.x : (int)threadIdx.x - 64 * W * group;
    f16* const keys[2] = {staged[group], staged[group] + KSIZE};
    f16* const values[2] = {staged[group] + 2 * KSIZE, staged[group] + 2 * KSIZE + VSIZE};
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lane = threadIdx.x & 63;
    const int n = lane & 31, h = lane >> 5;
    int item = blockIdx.x;
    const int split = item % a.splits;
    item /= a.splits;
    const int hk = item % a.kv_heads;
    item /= a.kv_heads;
    // the last rows, which see the most slots, are dispatched first
    const int tile = a.row_tiles - 1 - item % a.row_tiles, b = item / a.row_tiles;
    const int rows = a.tokens * a.group, row0 = tile * 32 * W, wave0 = row0 + 32 * wave;

    const uint8_t* kc = a.k_codes + b * a.kb + hk * a.kh;
    const uint8_t* vc = a.v_codes + b * a.vb + hk * a.vh;
    const float* ks = a.k_scales + b * a.ksb + hk * a.ksh;
    const float* vs = a.v_scales + b * a.vsb + hk * a.vsh;

    u32x4 kr[KL];
    uint32_t vr[8];
    const int vt = tid & (64 * VW - 1);
    const int vgroup = vt / (D / 4), vdim = vt % (D / 4);   // 8 slots, 4 dims of the values
    const bool loads_keys = KW == W || wave < KW, loads_values = VW == W || wave >= W - VW;
    // one uniform base and a 32-bit offset a load, at most that of the row of slot
    // `limit` (tiles past it read its tile's rows again) and of the tile's last
    // row: `limit` may lie more than 2^32 bytes behind the tile
    auto last_row = [&](int tile_at, int limit) { return (uint32_t)min(limit - tile_at * KT, KT - 1) * D; };
    auto load_keys = [&](int tile_at, int limit) {
        if (!loads_keys) return;
        tile_at = min(tile_at, limit / KT);
        const uint8_t* tile0 = kc + (int64_t)tile_at * (KT * D);
        const uint32_t most = last_row(tile_at, limit) + 16 * (tid % (D / 16));
#pragma unroll
        for (int i = 0; i < KL; ++i)
            kr[i] = *reinterpret_cast<const u32x4*>(tile0 + min((uint32_t)(16 * (tid + 64 * W * i)), most));
    };
    const uint32_t value0 = (16 * (vgroup >> 1) + 4 * (vgroup & 1)) * D + 4 * vdim;
    auto load_values = [&](int tile_at, int limit) {
        if (!loads_values) return;
        tile_at = min(tile_at, limit / KT);
        const uint8_t* tile0 = vc + (int64_t)tile_at * (KT * D);
        const uint32_t most = last_row(tile_at, limit) + 4 * vdim;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            vr[i] = *reinterpret_cast<const uint32_t*>(tile0 + min(value0 + (8 * (i >> 2) + (i & 3)) * D, most));
    };
#pragma unroll
    for (int i = 0; i < KL; ++i) kr[i] = (u32x4){0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < 8; ++i) vr[i] = 0;
    // the first tile of the first share does not depend on the sequence's length
    // and is requested before `start` has arrived (the other shares read the
    // first rows here and their own below)
    load_keys(split == 0 ? group : 0, (int)a.slots - 1);
    load_values(split == 0 ? group : 0, (int)a.slots - 1);

    const Seen seen = seen_of(a, b);
    const int end = seen_end(a, seen, row0, 32 * W);
    const int last_slot = max(end - 1, 0);
    const int tiles = (end + KT - 1) / KT;
    const Shares shares = shares_of(tiles, a.splits, a.least);
    if (split > 0 && split >= shares.count) return;
    if (split > 0) {
        load_keys(split * shares.size + group, last_slot);
        load_values(split * shares.size + group, last_slot);
    }
    const int first = split * shares.size + group, stop = min(tiles, (split + 1) * shares.size);

    const int r = min(wave0 + n, rows - 1);
    const int t = r / a.group, g = r - t * a.group;
    u32x4 qr[D / 16];
    {
        const uint16_t* q = a.q + b * a.qb + t * a.qt + (hk * a.group + g) * a.qh;
#pragma unroll
        for (int s = 0; s < D / 16; ++s) qr[s] = load8(q + 16 * s + 8 * h, a.vec);
    }
    const int64_t p = seen.start + t;
    const bool inside = t < seen.count && p >= 0 && p < a.slots;
    const int last = inside ? (int)p : -1;
    // slots from wave_end on are hidden from all rows of the wavefront; below wave_all no row needs a mask
    const int wave_end = seen_end(a, seen, wave0, 32);
    const int64_t p_first = seen.start + min(wave0, rows - 1) / a.group;
    const bool all_inside = wave0 + 32 <= rows && (wave0 + 31) / a.group < seen.count && p_first >= 0;
    const int wave_all = all_inside ? (int)min(p_first, a.slots - 1) + 1 : 0;

    // the scales of a tile's keys and values, 16 slots a lane (vector loads: scalar
    // ones share their counter with LDS, whose reads would wait for them)
    const float* scale_row = lane & (2 * KN) ? vs : ks;
    auto load_scales = [&](int tile_at) {
        return scale_row[min(tile_at * KT + 16 * (lane & (2 * KN - 1)), last_slot) >> a.block_log];
    };
    float scales = load_scales(first), scales_next = load_scales(first + KS);
    auto stage_keys = [&](f16* to) {
        if (!loads_keys) return;
#pragma unroll
        for (int i = 0; i < KL; ++i) {
            const int u = tid + 64 * W * i;
            f16x8* dst = reinterpret_cast<f16x8*>(to + (u / (D / 16)) * KROW + 16 * (u % (D / 16)));
            dst[0] = decode8<CODES>(kr[i][0], kr[i][1]);
            dst[1] = decode8<CODES>(kr[i][2], kr[i][3]);
        }
    };
    auto stage_values = [&](f16* to, int tile_at) {
        if (!loads_values) return;
        if ((tile_at + 1) * KT > end) {   // rows behind the last slot may hold anything
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (tile_at * KT + 16 * (vgroup >> 1) + 8 * (i >> 2) + 4 * (vgroup & 1) + (i & 3) >= end) vr[i] = 0;
        }
        // dim 4 v + d in row d D / 4 + v: neighbouring lanes write neighbouring rows
        f16x8 value[4];
        transpose8<CODES>(vr, value);
#pragma unroll
        for (int d = 0; d < 4; ++d)
            *reinterpret_cast<f16x8*>(to + (d * (D / 4) + vdim) * VROW + 8 * vgroup) = value[d];
    };
    float row_scale = a.scale * kLog2e * query_to_f16<TYPE>(qr, half_pair_max);
    // the largest score of a block is that of its largest product, and a masked
    // one stays -inf: a negative scale goes to q, and a factor too small to keep
    // its product with a scale of 2^-40 normal is raised (queries, codes and scales
    // at their ends then make scores of 2^-13, where they were to be smaller still)
    if (a.scale < 0.0f) {
        row_scale = -row_scale;
#pragma unroll
        for (int s = 0; s < D / 16; ++s) qr[s] ^= 0x80008000u;
    }
    row_scale = fmaxf(row_scale, 0x1p-86f);
    float run_max = -__builtin_inff(), run_sum = 0.0f;
    f32x16 acc[D / 32];
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[d][i] = 0.0f;

    // A tile's products go in 2 KN parts of P instructions each, so that those
    // of the next scores lie between the exponentials and the products of the
    // present weights. Fragments are read a part ahead; across kOrder only
    // vector instructions may be scheduled.
    constexpr int kOrder = 0x406, P = D / 32;
    f16x8 key[P], value[P];
    auto read_keys = [&](const f16* from, int part) {
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int m = P * part + i;
            key[i] = *reinterpret_cast<const f16x8*>(from + (32 * (m % KN) + n) * KROW + 16 * (m / KN) + 8 * h);
        }
    };
    auto products = [&](f16x8 (&q)[D / 16], int part, f32x16 (&to)[KN]) {   // of the scores
        if (part == 0) {
#pragma unroll
            for (int k = 0; k < KN; ++k)
#pragma unroll
                for (int i = 0; i < 16; ++i) to[k][i] = 0.0f;
        }
        __builtin_amdgcn_sched_barrier(kOrder);
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int m = P * part + i;
            to[m % KN] = __builtin_amdgcn_mfma_f32_32x32x16_f16(key[i], q[m / KN], to[m % KN], 0, 0, 0);
        }
        __builtin_amdgcn_sched_barrier(kOrder);
    };
    f16x8 q[D / 16];
#pragma unroll
    for (int s = 0; s < D / 16; ++s) q[s] = __builtin_bit_cast(f16x8, qr[s]);

    // Tile `at` of the loop has its scores in st and its values in LDS, the next
    // tile its keys: the next scores are formed while the softmax runs on the
    // present ones, and the codes of the keys after next and of the next values
    // are decoded while the present weights are multiplied.
    stage_keys(keys[0]);
    stage_values(values[0], first);
    load_keys(first + KS, last_slot);
    load_values(first + KS, last_slot);
    __syncthreads();
    f32x16 st[KN], next[KN];
#pragma unroll
    for (int x = 0; x < 2 * KN; ++x) {
        read_keys(keys[0], x);
        products(q, x, st);
    }
    stage_keys(keys[1]);
    load_keys(first + 2 * KS, last_slot);
    __syncthreads();
    auto tile_step = [&](int at, int now, f32x16 (&st)[KN], f32x16 (&next)[KN]) {
        const int slot0 = at * KT;
        if (slot0 < wave_end && (KS == 1 || at < stop)) {   // every wavefront meets the same barriers
            float mul[2 * KN], vex[2 * KN], vinv[2 * KN];
#pragma unroll
            for (int x = 0; x < 2 * KN; ++x) {
                const int bits = __builtin_bit_cast(int, scales);
                const int e = exponent_of(__builtin_bit_cast(float, __builtin_amdgcn_readlane(bits, 2 * KN + x)));
                mul[x] = row_scale * __builtin_bit_cast(float, __builtin_amdgcn_readlane(bits, x));
                vex[x] = (float)e;
                vinv[x] = exp2_int(-e);
            }
            if (slot0 + KT > wave_all) {
#pragma unroll
                for (int k = 0; k < KN; ++k)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (slot0 + 32 * k + 8 * (i >> 2) + 4 * h + (i & 3) > last) st[k][i] = -__builtin_inff();
            }
            read_keys(keys[now ^ 1], 0);
            float mx = -__builtin_inff();
#pragma unroll
            for (int x = 0; x < 2 * KN; ++x) {
                float top = st[x >> 1][8 * (x & 1)];
#pragma unroll
                for (int i = 1; i < 8; ++i) top = larger(top, st[x >> 1][8 * (x & 1) + i]);
                mx = larger(mx, __builtin_fmaf(top, mul[x], vex[x]));
            }
            mx = half_pair_max(mx);
            stage_keys(keys[now]);
            stage_values(values[now ^ 1], at + KS);
            load_keys(at + 3 * KS, last_slot);
            load_values(at + 2 * KS, last_slot);
            if (__any(mx - run_max > kMost)) {
                mx = reference(mx, run_max);
                const float rescale = mx == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(run_max - mx);
                run_max = mx;
                run_sum *= rescale;
#pragma unroll
                for (int d = 0; d < D / 32; ++d) acc[d] *= rescale;
            }
            const float base = run_max == -__builtin_inff() ? 0.0f : run_max;   // no slot of the row seen yet
#pragma unroll
            for (int x = 0; x < 2 * KN; ++x) {
#pragma unroll
                for (int d = 0; d < P; ++d)
                    value[d] = *reinterpret_cast<const f16x8*>(values[now] + (32 * d + n) * VROW + 16 * x + 8 * h);
                products(q, x, next);   // of no use past the last tile
                if (x + 1 < 2 * KN) read_keys(keys[now ^ 1], x + 1);
                const float shift = vex[x] - base;
                float sum = 0.0f;
                u32x4 packed;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float lo = __builtin_amdgcn_exp2f(__builtin_fmaf(st[x >> 1][8 * (x & 1) + 2 * i], mul[x], shift));
                    const float hi = __builtin_amdgcn_exp2f(__builtin_fmaf(st[x >> 1][8 * (x & 1) + 2 * i + 1], mul[x], shift));
                    // summed before the rounding: where values differ in scale, fp16 drops small
                    // weights of small values that hold most of the sum
                    sum += lo + hi;
                    packed[i] = as_u32((f16x2){(f16)lo, (f16)hi});
                }
                run_sum = __builtin_fmaf(sum, vinv[x], run_sum);
                __builtin_amdgcn_sched_barrier(kOrder);
#pragma unroll
                for (int d = 0; d < P; ++d)
                    acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(value[d], __builtin_bit_cast(f16x8, packed), acc[d],
                                                                    0, 0, 0);
                __builtin_amdgcn_sched_barrier(kOrder);
            }
        } else {
            stage_keys(keys[now]);
            stage_values(values[now ^ 1], at + KS);
            load_keys(at + 3 * KS, last_slot);
            load_values(at + 2 * KS, last_slot);
        }
        scales = scales_next;
        scales_next = load_scales(at + 2 * KS);
        __syncthreads();
    };
    // two tiles a round, so that the scores change places without copies
    // (a group without a tile in a round takes part in its barriers: such tiles
    // lie past the wavefront's last slot or are masked out whole)
    for (int at = first; at - group < stop; at += 2 * KS) {
        tile_step(at, 0, st, next);
        if (at - group + KS < stop) tile_step(at + KS, 1, next, st);
    }

    run_sum = half_pair_sum(run_sum);
    if constexpr (KS > 1) {   // the groups' states joined in the first (all tiles are used)
        constexpr int A = D / 2;   // outputs of a lane
        float* const other = reinterpret_cast<float*>(staged) + (A + 2) * 64 * wave + lane;
        static_assert((A + 2) * 64 * W * sizeof(float) <= sizeof(staged), "the outputs fit the tiles' memory");
        if (group == 1) {
            other[0] = run_max;
            other[64] = run_sum;
#pragma unroll
            for (int i = 0; i < A; ++i) other[64 * (2 + i)] = acc[i >> 4][i & 15];
        }
        __syncthreads();
        if (group == 1) return;
        const float max1 = other[0], top = fmaxf(run_max, max1);
        const float base = top == -__builtin_inff() ? 0.0f : top;
        const float f0 = __builtin_amdgcn_exp2f(run_max - base), f1 = __builtin_amdgcn_exp2f(max1 - base);
        run_max = top;
        run_sum = run_sum * f0 + other[64] * f1;
#pragma unroll
        for (int i = 0; i < A; ++i) acc[i >> 4][i & 15] = acc[i >> 4][i & 15] * f0 + other[64 * (2 + i)] * f1;
    }
    // R only grows: what a large one before the last has left is multiplied by 0, and shows if it is not finite
    float finite = 0.0f;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) finite = __builtin_fmaf(acc[d][i], 0.0f, finite);
    if (__any(fabsf(run_max) < __builtin_inff() && (fabsf(run_max) >= kLarge || finite != 0.0f))) {
        for (int row = wave0; row < min(wave0 + 32, rows); ++row)
            attend_row<D, CODES, TYPE>(a, seen, b, hk, row, (int64_t)split * shares.size * KT, (int64_t)stop * KT,
                                       shares.count > 1 ? split : -1);
        return;
    }
    if (wave0 + n >= rows) return;
    const int64_t at = ((int64_t)b * a.tokens + t) * a.heads + hk * a.group + g;
    // Row x of the values in LDS is dim 4 (x mod D / 4) + x / (D / 4), and acc[d][i]
    // is row 32 d + 8 (i >> 2) + 4 h + (i & 3): the v-th of the D / 8 runs of four
    // dims that a lane holds lies D / 4 rows apart.
    auto place = [](int v) { return 32 * (v >> 4) + 8 * ((v >> 2) & 3) + (v & 3); };   // its first row, without 4 h
    auto dim_of = [&](int v) { return 4 * (place(v) + 4 * h); };
    auto four = [&](int v) {
        f32x4 x;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int row = place(v) + e * (D / 4);
            x[e] = acc[row >> 5][4 * ((row >> 3) & 3) + (row & 3)];
        }
        return x;
    };
    if (shares.count > 1) {
        const int64_t sp = at * a.splits + split;
        if (h == 0) a.states[sp] = make_float2(run_max, run_sum);
        float* o = a.partial + sp * D;
#pragma unroll
        for (int v = 0; v < D / 8; ++v) {
            const f32x4 x = four(v);
            *reinterpret_cast<f32x4*>(o + dim_of(v)) = x;
        }
        return;
    }
    const bool padding = t >= seen.count;
    const float inv = padding ? 0.0f : inside ? 1.0f / run_sum : __builtin_nanf("");
    uint16_t* o = a.out + at * D;
#pragma unroll
    for (int v = 0; v < D / 8; ++v) {
        f32x4 x = four(v) * inv;
        if (padding) x = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
        store4<TYPE>(o + dim_of(v), x[0], x[1], x[2], x[3]);
    }
}

}  // namespace w4a16

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
