// Thin libtorch shim over the W4A16 C ABI: registers the torch ops
// w4a16::linear and w4a16::dequantize with the schemas of reference
// csrc/int4_linear.cpp:16-23 and w4a16::quantize (the reference quantizes in
// torch ops), implemented on the CUDA dispatch key (which is the HIP device on
// PyTorch-ROCm), and exposes an empty Python module so that importing the
// extension registers the ops (reference csrc/int4_linear.cpp:30). The ops of
// the 8-bit key/value cache (w4a16::rotary, kv_write, rotary_kv_write,
// kv_read, kv_attention, kv_shared_attention, kv_fork, kv_reorder) map tensors
// onto w4a16_kv.h and w4a16::sample onto w4a16_sample.h in the same way.
//
// Tensor-level checks use the reference's messages (reference
// csrc/int4_linear_kernel.cu:646-691, :809-841); shape relations and launches
// go through the C ABI. The output comes from the caching allocator on the
// activations' device and the work is enqueued on the current stream, so the
// op is graph-capture safe.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/library.h>

#include <cmath>
#include <type_traits>

#include "w4a16_hip.h"
#include "w4a16_kv.h"
#include "w4a16_sample.h"

namespace {

void* current_stream(const at::Device& device) {
    return static_cast<void*>(c10::hip::getCurrentHIPStream(device.index()).stream());
}

at::Tensor linear(const at::Tensor& activations, const at::Tensor& packed_weights, const at::Tensor& scales,
                  int64_t group_size) {
    TORCH_CHECK(activations.is_cuda(), "activations must be a CUDA tensor");
    TORCH_CHECK(packed_weights.is_cuda(), "packed_weights must be a CUDA tensor");
    TORCH_CHECK(scales.is_cuda(), "scales must be a CUDA tensor");
    TORCH_CHECK(activations.device() == packed_weights.device() && activations.device() == scales.device(),
                "all inputs must be on the same CUDA device");
    TORCH_CHECK(activations.scalar_type() == at::kHalf, "activations must have dtype torch.float16");
    TORCH_CHECK(packed_weights.scalar_type() == at::kByte, "packed_weights must have dtype torch.uint8");
    TORCH_CHECK(scales.scalar_type() == at::kHalf, "scales must have dtype torch.float16");
    TORCH_CHECK(activations.dim() == 2, "activations must have shape [M, K]");
    TORCH_CHECK(packed_weights.dim() == 2, "packed_weights must have shape [N, K / 2]");
    TORCH_CHECK(scales.dim() == 2, "scales must have shape [N, K / group_size]");
    TORCH_CHECK(activations.is_contiguous(), "activations must be contiguous");
    TORCH_CHECK(packed_weights.is_contiguous(), "packed_weights must be contiguous");
    TORCH_CHECK(scales.is_contiguous(), "scales must be contiguous");

    int rc = w4a16_check_linear_shapes(activations.size(0), activations.size(1), packed_weights.size(0),
                                       packed_weights.size(1), scales.size(0), scales.size(1), group_size);
    TORCH_CHECK(rc == W4A16_OK, w4a16_last_error());

    const int64_t M = activations.size(0);
    const int64_t K = activations.size(1);
    const int64_t N = packed_weights.size(0);
    const c10::DeviceGuard guard(activations.device());
    at::Tensor output = at::empty({M, N}, activations.options());
    if (M * N == 0) return output;

    void* const stream = current_stream(activations.device());
    if (M > 16) {   // prompt rows: no form of theirs has partial sums, so nothing of the library's scratch is used
        rc = w4a16_linear_noalloc_f16(activations.data_ptr(), packed_weights.data_ptr<uint8_t>(), scales.data_ptr(),
                                      output.data_ptr(), M, N, K, group_size, stream);
        TORCH_CHECK(rc == W4A16_OK, w4a16_last_error());
        return output;
    }
    // partial sums of the split-K kernel, from the caching allocator (so the
    // op stays graph-capture safe)
    const int64_t ws_bytes = w4a16_linear_workspace_bytes(M, N, K, group_size);
    at::Tensor workspace;
    if (ws_bytes > 0) workspace = at::empty({(ws_bytes + 3) / 4}, activations.options().dtype(at::kFloat));
    rc = w4a16_linear_ws_f16(activations.data_ptr(), packed_weights.data_ptr<uint8_t>(), scales.data_ptr(),
                             output.data_ptr(), M, N, K, group_size, ws_bytes > 0 ? workspace.data_ptr() : nullptr,
                             ws_bytes, stream);
    TORCH_CHECK(rc == W4A16_OK, w4a16_last_error());
    return output;
}

at::Tensor dequantize(const at::Tensor& packed_weights, const at::Tensor& scales, int64_t group_size) {
    TORCH_CHECK(packed_weights.is_cuda(), "packed_weights must be a CUDA tensor");
    TORCH_CHECK(scales.is_cuda(), "scales must be a CUDA tensor");
    TORCH_CHECK(packed_weights.device() == scales.device(),
                "packed_weights and scales must be on the same CUDA device");
    TORCH_CHECK(packed_weights.scalar_type() == at::kByte, "packed_weights must have dtype torch.uint8");
    TORCH_CHECK(scales.scalar_type() == at::kHalf, "scales must have dtype torch.float16");
    TORCH_CHECK(packed_weights.dim() == 2, "packed_weights must have shape [N, K / 2]");
    TORCH_CHECK(scales.dim() == 2, "scales must have shape [N, K / group_size]");
    TORCH_CHECK(packed_weights.is_contiguous(), "packed_weights must be contiguous");
    TORCH_CHECK(scales.is_contiguous(), "scales must be contiguous");

    int rc = w4a16_check_dequantize_shapes(packed_weights.size(0), packed_weights.size(1), scales.size(0),
                                           scales.size(1), group_size,
                                           reinterpret_cast<uint64_t>(packed_weights.data_ptr()));
    TORCH_CHECK(rc == W4A16_OK, w4a16_last_error());

    const int64_t N = packed_weights.size(0);
    const int64_t K = packed_weights.size(1) * 2;
    const c10::DeviceGuard guard(packed_weights.device());
    at::Tensor weights = at::empty({N, K}, packed_weights.options().dtype(at::kHalf));
    if (N * K == 0) return weights;
    rc = w4a16_dequantize_f16(packed_weights.data_ptr<uint8_t>(), scales.data_ptr(), weights.data_ptr(), N, K,
                              group_size, current_stream(packed_weights.device()));
    TORCH_CHECK(rc == W4A16_OK, w4a16_last_error());
    return weights;
}

// Weights [N, K] -> (packed uint8 [N, K / 2], scales fp16 [N, K / G]); the
// caller (nibble_amd/quantization.py) has made the quantizer's own checks.
std::tuple<at::Tensor, at::Tensor> quantize(const at::Tensor& weights, int64_t group_size) {
    TORCH_CHECK(weights.is_cuda(), "weights must be a CUDA tensor");
    TORCH_CHECK(weights.scalar_type() == at::kHalf || weights.scalar_type() == at::kFloat,
                "weights must have dtype torch.float16 or torch.float32");
    TORCH_CHECK(weights.dim() == 2 && weights.is_contiguous(), "weights must be contiguous with shape [N, K]");
    TORCH_CHECK(group_size > 0 && weights.size(1) % group_size == 0, "K must be divisible by group_size");
    const int64_t N = weights.size(0);
    const int64_t K = weights.size(1);
    const c10::DeviceGuard guard(weights.device());
    at::Tensor packed = at::empty({N, K / 2}, weights.options().dtype(at::kByte));
    at::Tensor scales = at::empty({N, K / group_size}, weights.options().dtype(at::kHalf));
    const int rc = w4a16_quantize_pack(weights.data_ptr(), (int)weights.element_size(), packed.data_ptr<uint8_t>(),
                                       scales.data_ptr(), N, K, group_size, current_stream(weights.device()));
    TORCH_CHECK(rc == W4A16_OK, w4a16_last_error());
    return {packed, scales};
}

// ------------------------------------------------------------ the 8-bit key/value cache

int row_type(const at::Tensor& x, const char* name) {
    TORCH_CHECK(x.scalar_type() == at::kHalf || x.scalar_type() == at::kBFloat16, name,
                " must have dtype torch.float16 or torch.bfloat16");
    return x.scalar_type() == at::kHalf ? W4A16_FP16 : W4A16_BF16;
}

// A dimension of one element has no step.
int64_t stride_of(const at::Tensor& x, int64_t dim) { return x.size(dim) > 1 ? x.stride(dim) : 0; }

// Token rows [batch, tokens, heads, head_dim].
w4a16_kv_rows rows_of(const at::Tensor& x, const char* name) {
    TORCH_CHECK(x.is_cuda(), name, " must be a CUDA tensor");
    TORCH_CHECK(!x.requires_grad(), name, " must not require grad");
    TORCH_CHECK(x.dim() == 4, name, " must have shape [batch, tokens, heads, head_dim]");
    TORCH_CHECK(x.size(3) <= 1 || x.stride(3) == 1, name, " must be contiguous in its last dimension");
    return {x.data_ptr(), stride_of(x, 0), stride_of(x, 1), stride_of(x, 2)};
}

int code_type(const at::Tensor& codes, const char* name) {
    TORCH_CHECK(codes.scalar_type() == at::kChar || codes.scalar_type() == at::kFloat8_e4m3fn, name,
                " must have dtype torch.int8 or torch.float8_e4m3fn");
    return codes.scalar_type() == at::kChar ? W4A16_KV_INT8 : W4A16_KV_FP8;
}

// Slots of a scale: the block size of which `blocks` cover `slots` (there is
// one at most past one block; one block is any size that holds the slots).
int64_t block_of(int64_t slots, int64_t blocks) {
    for (int64_t block = 16; block <= 128; block *= 2)
        if ((slots + block - 1) / block == blocks) return block;
    return 0;
}

w4a16_kv_codes codes_of(const at::Tensor& codes, const at::Tensor& scales, const char* name) {
    TORCH_CHECK(codes.is_cuda() && scales.is_cuda(), name, " codes and scales must be CUDA tensors");
    TORCH_CHECK(codes.device() == scales.device(), name, " codes and scales must be on the same CUDA device");
    TORCH_CHECK(scales.scalar_type() == at::kFloat, name, " scales must have dtype torch.float32");
    TORCH_CHECK(!codes.requires_grad() && !scales.requires_grad(), name, " codes and scales must not require grad");
    TORCH_CHECK(codes.dim() == 4, name, " codes must have shape [batch, kv_heads, slots, head_dim]");
    TORCH_CHECK(scales.dim() == 3 && scales.size(0) == codes.size(0) && scales.size(1) == codes.size(1), name,
                " scales must have shape [batch, kv_heads, blocks]");
    TORCH_CHECK((codes.size(3) <= 1 || codes.stride(3) == 1) && (codes.size(2) <= 1 || codes.stride(2) == codes.size(3)),
                name, " codes must be contiguous in slots and head_dim");
    TORCH_CHECK(scales.size(2) <= 1 || scales.stride(2) == 1, name, " scales must be contiguous in blocks");
    TORCH_CHECK(block_of(codes.size(2), scales.size(2)) != 0 || codes.size(2) == 0, name,
                " scales must hold one scale for every 16, 32, 64 or 128 slots");
    return {codes.data_ptr(), scales.data_ptr<float>(), stride_of(codes, 0), stride_of(codes, 1),
            stride_of(scales, 0), stride_of(scales, 1)};
}

struct Cache {
    w4a16_kv_cache abi;
    at::Device device;
};

Cache cache_of(const at::Tensor& k_codes, const at::Tensor& k_scales, const at::Tensor& v_codes,
               const at::Tensor& v_scales) {
    const w4a16_kv_codes k = codes_of(k_codes, k_scales, "key"), v = codes_of(v_codes, v_scales, "value");
    TORCH_CHECK(k_codes.device() == v_codes.device(), "keys and values must be on the same CUDA device");
    TORCH_CHECK(k_codes.scalar_type() == v_codes.scalar_type(), "key and value codes must have the same dtype");
    TORCH_CHECK(k_codes.sizes() == v_codes.sizes() && k_scales.sizes() == v_scales.sizes(),
                "key and value codes and scales must have the same shapes");
    return {{k, v, k_codes.size(0), k_codes.size(1), k_codes.size(2), k_codes.size(3),
             block_of(k_codes.size(2), k_scales.size(2)), code_type(k_codes, "codes")},
            k_codes.device()};
}

// Device int64 [batch]: a sequence's first position, or its count of tokens.
const int64_t* lengths_of(const at::Tensor& x, int64_t batch, const at::Device& device, const char* name) {
    TORCH_CHECK(x.is_cuda() && x.device() == device, name, " must be on the cache's CUDA device");
    TORCH_CHECK(x.scalar_type() == at::kLong, name, " must have dtype torch.int64");
    TORCH_CHECK(x.dim() == 1 && x.size(0) == batch && x.is_contiguous(), name, " must be contiguous with shape [batch]");
    return x.data_ptr<int64_t>();
}

const int64_t* counts_of(const c10::optional<at::Tensor>& counts, int64_t batch, const at::Device& device) {
    return counts.has_value() && counts->defined() ? lengths_of(*counts, batch, device, "counts") : nullptr;
}

void check_tables(const at::Tensor& cos, const at::Tensor& sin, const at::Device& device) {
    TORCH_CHECK(cos.is_cuda() && cos.device() == device && sin.is_cuda() && sin.device() == device,
                "cos and sin must be on the same CUDA device as the rows");
    TORCH_CHECK(!cos.requires_grad() && !sin.requires_grad(), "cos and sin must not require grad");
    TORCH_CHECK(cos.scalar_type() == at::kFloat && sin.scalar_type() == at::kFloat,
                "cos and sin must have dtype torch.float32");
    TORCH_CHECK(cos.dim() == 2 && cos.sizes() == sin.sizes() && cos.is_contiguous() && sin.is_contiguous(),
                "cos and sin must be contiguous with shape [positions, rotated dims / 2]");
}

// Rows of new tokens that go with a cache.
w4a16_kv_rows token_rows(const at::Tensor& x, const Cache& cache, int64_t tokens, int64_t heads, const char* name) {
    const w4a16_kv_rows rows = rows_of(x, name);
    TORCH_CHECK(x.device() == cache.device, name, " must be on the cache's CUDA device");
    TORCH_CHECK(x.size(0) == cache.abi.batch && x.size(1) == tokens && (heads < 0 || x.size(2) == heads) &&
                    x.size(3) == cache.abi.head_dim,
                name, " must have shape [batch, tokens, heads, head_dim] of the cache and of the other rows");
    return rows;
}

at::Tensor rotary(const at::Tensor& x, const at::Tensor& positions, const at::Tensor& cos, const at::Tensor& sin,
                  bool interleaved) {
    const at::Tensor wide = x.dim() == 3 ? x.unsqueeze(0) : x;
    TORCH_CHECK(wide.dim() == 4, "x must have shape [tokens, heads, head_dim] or [batch, tokens, heads, head_dim]");
    const w4a16_kv_rows rows = rows_of(wide, "x");
    const int type = row_type(x, "x");
    TORCH_CHECK(positions.is_cuda() && positions.device() == x.device(), "positions must be on the same CUDA device as x");
    TORCH_CHECK(positions.scalar_type() == at::kLong, "positions must have dtype torch.int64");
    const bool shared = positions.dim() == 1;   // by all sequences
    TORCH_CHECK((shared && positions.size(0) == wide.size(1)) ||
                    (positions.dim() == 2 && x.dim() == 4 && positions.size(0) == wide.size(0) &&
                     positions.size(1) == wide.size(1)),
                "positions must have shape [tokens] or [batch, tokens]");
    check_tables(cos, sin, x.device());
    const c10::DeviceGuard guard(x.device());
    at::Tensor out = at::empty(x.sizes(), x.options(), at::MemoryFormat::Contiguous);
    const int rc = w4a16_rotary(&rows, out.data_ptr(), wide.size(0), wide.size(1), wide.size(2), wide.size(3),
                                cos.data_ptr<float>(), sin.data_ptr<float>(), cos.size(0), 2 * cos.size(1),
                                positions.data_ptr<int64_t>(), shared ? 0 : positions.stride(0),
                                positions.stride(shared ? 0 : 1), interleaved, type, current_stream(x.device()));
    TORCH_CHECK(rc == W4A16_OK, w4a16_last_error());
    return out;
}

void kv_write(const at::Tensor& k, const at::Tensor& v, at::Tensor k_codes, at::Tensor k_scales, at::Tensor v_codes,
              at::Tensor v_scales, const at::Tensor& start, const c10::optional<at::Tensor>& counts) {
    const Cache cache = cache_of(k_codes, k_scales, v_codes, v_scales);
    TORCH_CHECK(k.dim() == 4, "k must have shape [batch, tokens, heads, head_dim]");
    const w4a16_kv_rows kr = token_rows(k, cache, k.size(1), cache.abi.kv_heads, "k");
    const w4a16_kv_rows vr = token_rows(v, cache, k.size(1), cache.abi.kv_heads, "v");
    const int type = row_type(k, "k");
    TORCH_CHECK(v.scalar_type() == k.scalar_type(), "k and v must have the same dtype");
    const int64_t* first = lengths_of(start, cache.abi.batch, cache.device, "start");
    const c10::DeviceGuard guard(cache.device);
    const int rc = w4a16_kv_write(&kr, &vr, k.size(1), &cache.abi, first,
                                  counts_of(counts, cache.abi.batch, cache.device), type, current_stream(cache.device));
    TORCH_CHECK(rc == W4A16_OK, w4a16_last_error());
}

at::Tensor rotary_kv_write(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& cos,
                           const at::Tensor& sin, at::Tensor k_codes, at::Tensor k_scales, at::Tensor v_codes,
                           at::Tensor v_scales, const at::Tensor& start, const c10::optional<at::Tensor>& counts,
                           bool interleaved) {
    const Cache cache = cache_of(k_codes, k_scales, v_codes, v_scales);
    TORCH_CHECK(q.dim() == 4, "q must have shape [batch, tokens, heads, head_dim]");
    const int64_t tokens = q.size(1);
    const w4a16_kv_rows qr = token_rows(q, cache, tokens, -1, "q");
    const w4a16_kv_rows kr = token_rows(k, cache, tokens, cache.abi.kv_heads, "k");
    const w4a16_kv_rows vr = token_rows(v, cache, tokens, cache.abi.kv_heads, "v");
    const int type = row_type(q, "q");
    TORCH_CHECK(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(),
                "q, k and v must have the same dtype");
    check_tables(cos, sin, cache.device);
    const int64_t* first = lengths_of(start, cache.abi.batch, cache.device, "start");
    const c10::DeviceGuard guard(cache.device);
    at::Tensor out = at::empty(q.sizes(), q.options(), at::MemoryFormat::Contiguous);
    const int rc = w4a16_rotary_kv_write(&qr, out.data_ptr(), q.size(2), &kr, &vr, tokens, cos.data_ptr<float>(),
                                         sin.data_ptr<float>(), cos.size(0), 2 * cos.size(1), interleaved, &cache.abi,
                                         first, counts_of(counts, cache.abi.batch, cache.device), type,
                                         current_stream(cache.device));
    TORCH_CHECK(rc == W4A16_OK, w4a16_last_error());
    return out;
}

at::Tensor kv_read(const at::Tensor& codes, const at::Tensor& scales, at::ScalarType dtype) {
    const w4a16_kv_codes side = codes_of(codes, scales, "the");
    const int type = code_type(codes, "codes");
    TORCH_CHECK(dtype == at::kHalf || dtype == at::kBFloat16 || dtype == at::kFloat,
                "dtype must be torch.float16, torch.bfloat16 or torch.float32");
    const c10::DeviceGuard guard(codes.device());
    at::Tensor out = at::empty(codes.sizes(), codes.options().dtype(dtype), at::MemoryFormat::Contiguous);
    if (out.numel() == 0) return out;
    const int rc = w4a16_kv_read(&side, out.data_ptr(), codes.size(0), codes.size(1), codes.size(2), codes.size(3),
                                 block_of(codes.size(2), scales.size(2)), type,
                                 dtype == at::kHalf ? W4A16_FP16 : dtype == at::kBFloat16 ? W4A16_BF16 : W4A16_FP32,
                                 current_stream(codes.device()));
    TORCH_CHECK(rc == W4A16_OK, w4a16_last_error());
    return out;
}

at::Tensor kv_attention(const at::Tensor& q, const at::Tensor& k_codes, const at::Tensor& k_scales,
                        const at::Tensor& v_codes, const at::Tensor& v_scales, const at::Tensor& start,
                        const c10::optional<at::Tensor>& counts, c10::optional<double> scale) {
    const Cache cache = cache_of(k_codes, k_scales, v_codes, v_scales);
    TORCH_CHECK(q.dim() == 4, "q must have shape [batch, tokens, heads, head_dim]");
    const int64_t tokens = q.size(1), heads = q.size(2);
    const w4a16_kv_rows qr = token_rows(q, cache, tokens, -1, "q");
    const int type = row_type(q, "q");
    const int64_t* first = lengths_of(start, cache.abi.batch, cache.device, "start");
    const c10::DeviceGuard guard(cache.device);
    at::Tensor out = at::empty(q.sizes(), q.options(), at::MemoryFormat::Contiguous);
    // partial results of shares of the slots, from the caching allocator (graph-capture safe)
    const int64_t ws_bytes = w4a16_kv_attention_workspace_bytes(cache.abi.batch, tokens, heads, cache.abi.kv_heads,
                                                                cache.abi.slots, cache.abi.head_dim);
    at::Tensor workspace;
    if (ws_bytes > 0) workspace = at::empty({(ws_bytes + 3) / 4}, q.options().dtype(at::kFloat));
    const int rc = w4a16_kv_attention(&qr, out.data_ptr(), tokens, heads, &cache.abi, first,
                                      counts_of(counts, cache.abi.batch, cache.device),
                                      (float)(scale.has_value() ? *scale : 1.0 / std::sqrt((double)cache.abi.head_dim)),
                                      type, ws_bytes > 0 ? workspace.data_ptr() : nullptr, ws_bytes,
                                      current_stream(cache.device));
    TORCH_CHECK(rc == W4A16_OK, w4a16_last_error());
    return out;
}

at::Tensor kv_shared_attention(const at::Tensor& q, const at::Tensor& prefix_k_codes, const at::Tensor& prefix_k_scales,
                               const at::Tensor& prefix_v_codes, const at::Tensor& prefix_v_scales,
                               const at::Tensor& prefix_lengths, const at::Tensor& k_codes, const at::Tensor& k_scales,
                               const at::Tensor& v_codes, const at::Tensor& v_scales, const at::Tensor& start,
                               const c10::optional<at::Tensor>& counts, c10::optional<double> scale) {
    const Cache prefix = cache_of(prefix_k_codes, prefix_k_scales, prefix_v_codes, prefix_v_scales);
    const Cache cache = cache_of(k_codes, k_scales, v_codes, v_scales);
    TORCH_CHECK(prefix.device == cache.device, "the prefix must be on the cache's CUDA device");
    TORCH_CHECK(q.dim() == 4, "q must have shape [batch, tokens, heads, head_dim]");
    const int64_t tokens = q.size(1), heads = q.size(2);
    const w4a16_kv_rows qr = token_rows(q, cache, tokens, -1, "q");
    const int type = row_type(q, "q");
    const int64_t* lengths = lengths_of(prefix_lengths, prefix.abi.batch, cache.device, "prefix_lengths");
    const int64_t* first = lengths_of(start, cache.abi.batch, cache.device, "start");
    const c10::DeviceGuard guard(cache.device);
    at::Tensor out = at::empty(q.sizes(), q.options(), at::MemoryFormat::Contiguous);
    // the shares of both sides, from the caching allocator (graph-capture safe)
    const int64_t ws_bytes = w4a16_kv_shared_attention_workspace_bytes(
        prefix.abi.batch, prefix.abi.slots, cache.abi.batch, tokens, heads, cache.abi.kv_heads, cache.abi.slots,
        cache.abi.head_dim);
    at::Tensor workspace;
    if (ws_bytes > 0) workspace = at::empty({(ws_bytes + 3) / 4}, q.options().dtype(at::kFloat));
    const int rc = w4a16_kv_shared_attention(
        &qr, out.data_ptr(), tokens, heads, &prefix.abi, lengths, &cache.abi, first,
        counts_of(counts, cache.abi.batch, cache.device),
        (float)(scale.has_value() ? *scale : 1.0 / std::sqrt((double)cache.abi.head_dim)), type,
        ws_bytes > 0 ? workspace.data_ptr() : nullptr, ws_bytes, current_stream(cache.device));
    TORCH_CHECK(rc == W4A16_OK, w4a16_last_error());
    return out;
}

void kv_fork(const at::Tensor& k_codes, const at::Tensor& k_scales, const at::Tensor& v_codes,
             const at::Tensor& v_scales, at::Tensor to_k_codes, at::Tensor to_k_scales, at::Tensor to_v_codes,
             at::Tensor to_v_scales, const at::Tensor& source, const at::Tensor& lengths) {
    Cache from = cache_of(k_codes, k_scales, v_codes, v_scales);
    Cache to = cache_of(to_k_codes, to_k_scales, to_v_codes, to_v_scales);
    TORCH_CHECK(from.device == to.device, "both caches must be on the same CUDA device");
    // slots that one scale covers may be of any block that holds them: the other cache tells which
    if (k_scales.size(2) == 1 && from.abi.slots <= to.abi.block) from.abi.block = to.abi.block;
    if (to_k_scales.size(2) == 1 && to.abi.slots <= from.abi.block) to.abi.block = from.abi.block;
    const int64_t* rows = lengths_of(source, to.abi.batch, to.device, "source");
    const int64_t* held = lengths_of(lengths, from.abi.batch, to.device, "lengths");
    const c10::DeviceGuard guard(to.device);
    const int rc = w4a16_kv_fork(&from.abi, &to.abi, rows, held, current_stream(to.device));
    TORCH_CHECK(rc == W4A16_OK, w4a16_last_error());
}

void kv_reorder(at::Tensor k_codes, at::Tensor k_scales, at::Tensor v_codes, at::Tensor v_scales,
                const at::Tensor& source, const at::Tensor& lengths) {
    const Cache cache = cache_of(k_codes, k_scales, v_codes, v_scales);
    const int64_t* rows = lengths_of(source, cache.abi.batch, cache.device, "source");
    const int64_t* held = lengths_of(lengths, cache.abi.batch, cache.device, "lengths");
    const c10::DeviceGuard guard(cache.device);
    const int rc = w4a16_kv_reorder(&cache.abi, rows, held, current_stream(cache.device));
    TORCH_CHECK(rc == W4A16_OK, w4a16_last_error());
}

// ------------------------------------------------------------ sampling

// One value a row, or none.
template <typename T>
const T* row_values(const c10::optional<at::Tensor>& x, int64_t rows, const at::Device& device, const char* name) {
    if (!x.has_value() || !x->defined()) return nullptr;
    constexpr bool whole = std::is_same<T, int64_t>::value;
    TORCH_CHECK(x->is_cuda() && x->device() == device, name, " must be on the same CUDA device as the logits");
    TORCH_CHECK(!x->requires_grad(), name, " must not require grad");
    TORCH_CHECK(x->scalar_type() == (whole ? at::kLong : at::kFloat), name, " must have dtype ",
                whole ? "torch.int64" : "torch.float32");
    TORCH_CHECK(x->dim() == 1 && x->size(0) == rows && x->is_contiguous(), name,
                " must be contiguous with shape [rows]");
    return x->template data_ptr<T>();
}

at::Tensor sample(const at::Tensor& logits, const at::Tensor& random, double temperature, int64_t top_k, double top_p,
                  double min_p, const c10::optional<at::Tensor>& temperatures,
                  const c10::optional<at::Tensor>& top_ks, const c10::optional<at::Tensor>& top_ps,
                  const c10::optional<at::Tensor>& min_ps) {
    TORCH_CHECK(logits.is_cuda(), "logits must be a CUDA tensor");
    TORCH_CHECK(logits.scalar_type() == at::kHalf || logits.scalar_type() == at::kBFloat16 ||
                    logits.scalar_type() == at::kFloat,
                "logits must have dtype torch.float16, torch.bfloat16 or torch.float32");
    TORCH_CHECK(!logits.requires_grad(), "logits must not require grad");
    TORCH_CHECK(logits.dim() == 2, "logits must have shape [rows, vocabulary]");
    TORCH_CHECK(logits.size(1) <= 1 || logits.stride(1) == 1, "logits must be contiguous in their last dimension");
    const int64_t rows = logits.size(0);
    const at::Device device = logits.device();
    const float* numbers = row_values<float>(random, rows, device, "random");
    TORCH_CHECK(numbers != nullptr || rows == 0, "random must have a value for every row");
    const w4a16_sample_settings settings{temperature, top_k, top_p, min_p,
                                         row_values<float>(temperatures, rows, device, "temperature"),
                                         row_values<int64_t>(top_ks, rows, device, "top_k"),
                                         row_values<float>(top_ps, rows, device, "top_p"),
                                         row_values<float>(min_ps, rows, device, "min_p")};
    const c10::DeviceGuard guard(device);
    at::Tensor tokens = at::empty({rows}, logits.options().dtype(at::kLong));
    const int type = logits.scalar_type() == at::kHalf       ? W4A16_FP16
                     : logits.scalar_type() == at::kBFloat16 ? W4A16_BF16
                                                             : W4A16_FP32;
    const int rc = w4a16_sample(logits.data_ptr(), rows, logits.size(1), stride_of(logits, 0), type, numbers, &settings,
                                tokens.data_ptr<int64_t>(), current_stream(device));
    TORCH_CHECK(rc == W4A16_OK, w4a16_last_error());
    return tokens;
}

}  // namespace

TORCH_LIBRARY(w4a16, m) {
    m.def("linear(Tensor activations, Tensor packed_weights, Tensor scales, int group_size) -> Tensor");
    m.def("dequantize(Tensor packed_weights, Tensor scales, int group_size) -> Tensor");
    m.def("quantize(Tensor weights, int group_size) -> (Tensor, Tensor)");
    m.def("rotary(Tensor x, Tensor positions, Tensor cos, Tensor sin, bool interleaved=False) -> Tensor");
    m.def("kv_write(Tensor k, Tensor v, Tensor(a!) k_codes, Tensor(b!) k_scales, Tensor(c!) v_codes, "
          "Tensor(d!) v_scales, Tensor start, Tensor? counts=None) -> ()");
    m.def("rotary_kv_write(Tensor q, Tensor k, Tensor v, Tensor cos, Tensor sin, Tensor(a!) k_codes, "
          "Tensor(b!) k_scales, Tensor(c!) v_codes, Tensor(d!) v_scales, Tensor start, Tensor? counts=None, "
          "bool interleaved=False) -> Tensor");
    m.def("kv_read(Tensor codes, Tensor scales, ScalarType dtype) -> Tensor");
    m.def("kv_attention(Tensor q, Tensor k_codes, Tensor k_scales, Tensor v_codes, Tensor v_scales, Tensor start, "
          "Tensor? counts=None, float? scale=None) -> Tensor");
    m.def("kv_shared_attention(Tensor q, Tensor prefix_k_codes, Tensor prefix_k_scales, Tensor prefix_v_codes, "
          "Tensor prefix_v_scales, Tensor prefix_lengths, Tensor k_codes, Tensor k_scales, Tensor v_codes, "
          "Tensor v_scales, Tensor start, Tensor? counts=None, float? scale=None) -> Tensor");
    m.def("kv_fork(Tensor k_codes, Tensor k_scales, Tensor v_codes, Tensor v_scales, Tensor(a!) to_k_codes, "
          "Tensor(b!) to_k_scales, Tensor(c!) to_v_codes, Tensor(d!) to_v_scales, Tensor source, Tensor lengths) -> ()");
    m.def("kv_reorder(Tensor(a!) k_codes, Tensor(b!) k_scales, Tensor(c!) v_codes, Tensor(d!) v_scales, "
          "Tensor source, Tensor lengths) -> ()");
    m.def("sample(Tensor logits, Tensor random, float temperature=1.0, int top_k=0, float top_p=1.0, "
          "float min_p=0.0, Tensor? temperatures=None, Tensor? top_ks=None, Tensor? top_ps=None, "
          "Tensor? min_ps=None) -> Tensor");
}

TORCH_LIBRARY_IMPL(w4a16, CUDA, m) {
    m.impl("linear", &linear);
    m.impl("dequantize", &dequantize);
    m.impl("quantize", &quantize);
    m.impl("rotary", &rotary);
    m.impl("kv_write", &kv_write);
    m.impl("rotary_kv_write", &rotary_kv_write);
    m.impl("kv_read", &kv_read);
    m.impl("kv_attention", &kv_attention);
    m.impl("kv_shared_attention", &kv_shared_attention);
    m.impl("kv_fork", &kv_fork);
    m.impl("kv_reorder", &kv_reorder);
    m.impl("sample", &sample);
}

static PyModuleDef w4a16_module = {PyModuleDef_HEAD_INIT, "_C", "W4A16 torch ops (registered on import)", -1,
                                   nullptr};

PyMODINIT_FUNC PyInit__C(void) { return PyModule_Create(&w4a16_module); }
