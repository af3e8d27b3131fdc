// Torch extension module `decoding_attn_cuda`: the call surface of the reference's binding
// (csrc/torch/decoding_torch.cpp:19-85) on top of this library's C ABI.
//
//   fwd(q, k, v_, o_, cu_seq_k, max_seq_k, dim_v, is_alibi) -> o      same positional signature and
//       checks as the reference's dmha_fwd (decoding_torch.cpp:19-80); v_ = None selects MLA.
//   dmha_fwd(q, k, v, cu_seq_k, max_seq_k, is_alibi, softmax_scale=None, out=None, return_lse=False, k_scale=1, v_scale=1)
//       (k, v may be torch.float8_e4m3fn: an FP8 cache standing for k * k_scale, v * v_scale)
//   dmla_fwd(q, kv, cu_seq_k, max_seq_k, dim_v=512, is_alibi=False, softmax_scale=None, out=None, return_lse=False)
//       the two named entry points with an explicit softmax scale; their defaults reproduce fwd().
//   merge_partials(part_o, part_lse, out_dtype) -> (o, lse)           LSE merge of key-range shards.
//   kv_cache_write(k, v, k_cache, v_cache, k_scale, v_scale, slots=None), kv_cache_read(...) -> (k, v),
//   quantized_fwd(q, k_cache, v_cache, k_scale, v_scale, cu_seq_k, ...) -> o: caches with a scale per (token, KV head).
//   shared_prefix_fwd(q, k_prefix, v_prefix, k, v, cu_seq_k, ...) -> o: decode of a batch whose sequences share a prefix.
//
// Differences from the reference, all on the safe side: a device guard on q's device (the
// reference takes none, so it only works on the current device), real row strides are passed down
// instead of assuming packed rows (decoding_attn.cpp:32-46), and library errors raise instead of
// terminating the process.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <array>
#include <cstring>
#include <optional>
#include <tuple>

#include "../../include/decoding_attn_b200.h"

namespace {

#define DA_CHECK_DEVICE(x) TORCH_CHECK(x.is_cuda(), #x " must be on CUDA")
#define DA_CHECK_SHAPE(x, ...) \
    TORCH_CHECK(x.sizes() == torch::IntArrayRef({__VA_ARGS__}), #x " must have shape (" #__VA_ARGS__ ")")
#define DA_CHECK_CONTIGUOUS(x) TORCH_CHECK(x.is_contiguous(), #x " must be contiguous")

struct Outputs {
    at::Tensor o;
    at::Tensor lse;
};

// Whether rows [tokens, heads, dim] share memory, as those of a tensor expanded over its tokens do (row stride 0, which
// the library takes for packed rows).
bool rows_overlap(const at::Tensor &x) { return x.dim() == 3 && x.size(0) > 1 && x.stride(0) < x.size(1) * x.size(2); }
at::Tensor own_rows(const at::Tensor &x) { return rows_overlap(x) ? x.contiguous() : x; }

Outputs run(const at::Tensor &q_, const at::Tensor &k_, const std::optional<at::Tensor> &v_,
            const std::optional<at::Tensor> &o_, const at::Tensor &cu_seq_k, int64_t max_seq_k, int64_t dim_v,
            bool is_alibi, std::optional<double> softmax_scale, bool want_lse, const at::Tensor *block_table = nullptr,
            int64_t page_size = 0, double k_scale = 1.0, double v_scale = 1.0) {
    const at::Tensor q = own_rows(q_), k = own_rows(k_);
    auto q_dtype = q.dtype();
    TORCH_CHECK(q_dtype == torch::kFloat16 || q_dtype == torch::kBFloat16,
                "Decoding-Attention only support FP16 and BF16 data type");
    const bool is_bf16 = q_dtype == torch::kBFloat16;
    // An FP8 e4m3 cache (k and v both) is an extension; the reference requires the dtype of q
    // (csrc/torch/decoding_torch.cpp:28, :57).
    // A quantised cache (k and v both) is an extension: FP8 e4m3, or int8 (torch.int8); int4 goes through the C ABI.
    const bool int8_cache = k.scalar_type() == at::kChar;
    const bool fp8_cache = k.scalar_type() == at::kFloat8_e4m3fn || int8_cache;
    TORCH_CHECK(fp8_cache || k.dtype() == q_dtype, "query and key must have the same dtype");
    TORCH_CHECK(cu_seq_k.dtype() == torch::kInt32, "cu_seq_k must have dtype int32");

    DA_CHECK_DEVICE(q);
    DA_CHECK_DEVICE(k);
    DA_CHECK_DEVICE(cu_seq_k);
    TORCH_CHECK(k.device() == q.device() && cu_seq_k.device() == q.device(), "all tensors must be on one device");
    TORCH_CHECK(q.dim() == 3 && k.dim() == 3, "query and key must be 3-D");

    TORCH_CHECK(q.stride(-1) == 1, "query must have contiguous last dimension");
    TORCH_CHECK(k.stride(-1) == 1, "key must have contiguous last dimension");
    DA_CHECK_CONTIGUOUS(cu_seq_k);

    const int64_t batch = cu_seq_k.numel() - 1;
    const int64_t total_q = q.size(0);
    const int64_t head_q = q.size(1);
    const int64_t dim = q.size(2);
    const int64_t total_k = k.size(0);
    const int64_t head_k = k.size(1);
    TORCH_CHECK(batch > 0, "batch size must be positive");
    TORCH_CHECK(total_q == batch, "one query token per sequence: q.size(0) must equal cu_seq_k.numel() - 1");
    TORCH_CHECK(dim <= 576, "dim should be at most 576");
    TORCH_CHECK(dim_v <= 512, "dim_v should be at most 512");
    TORCH_CHECK(head_q % head_k == 0, "number of heads in key/value must divide number of heads in query");

    DA_CHECK_SHAPE(q, total_q, head_q, dim);
    DA_CHECK_SHAPE(k, total_k, head_k, dim);
    DA_CHECK_SHAPE(cu_seq_k, batch + 1);
    TORCH_CHECK(q.stride(1) == dim && k.stride(1) == dim, "heads must be contiguous inside a token row");

    const at::cuda::CUDAGuard guard(q.device());
    auto stream = at::cuda::getCurrentCUDAStream().stream();

    da_decode_args_t a;
    std::memset(&a, 0, sizeof(a));
    a.struct_size = sizeof(a);
    a.is_bf16 = is_bf16;
    a.is_alibi = is_alibi;
    a.q = q.data_ptr();
    a.k = k.data_ptr();
    a.q_row_stride = q.stride(0);
    a.k_row_stride = k.stride(0);

    at::Tensor v;  // (kept until the launch: it may be a copy)
    if (v_.has_value()) {
        v = own_rows(v_.value());
        TORCH_CHECK(v.dtype() == k.dtype(), fp8_cache ? "key and value must have the same quantised dtype" : "query and value must have the same dtype");
        DA_CHECK_DEVICE(v);
        TORCH_CHECK(v.device() == q.device(), "all tensors must be on one device");
        TORCH_CHECK(v.stride(-1) == 1, "value must have contiguous last dimension");
        DA_CHECK_SHAPE(v, total_k, head_k, dim_v);
        TORCH_CHECK(v.stride(1) == dim_v, "heads must be contiguous inside a token row");
        a.v = v.data_ptr();
        a.v_row_stride = v.stride(0);
    }

    Outputs out;
    if (o_.has_value()) {
        out.o = o_.value();
        TORCH_CHECK(out.o.dtype() == q_dtype, "Output must have the same dtype as inputs");
        DA_CHECK_DEVICE(out.o);
        TORCH_CHECK(out.o.device() == q.device(), "all tensors must be on one device");
        TORCH_CHECK(out.o.stride(-1) == 1, "Output tensor must have contiguous last dimension");
        DA_CHECK_SHAPE(out.o, total_q, head_q, dim_v);
        TORCH_CHECK(out.o.stride(1) == dim_v, "heads must be contiguous inside a token row");
        TORCH_CHECK(!rows_overlap(out.o), "Output tensor must have rows of its own for every sequence");
    } else {
        out.o = torch::empty({total_q, head_q, dim_v}, q.options());
    }
    a.o = out.o.data_ptr();
    a.o_row_stride = out.o.stride(0);
    if (want_lse) {
        out.lse = torch::empty({total_q, head_q}, q.options().dtype(torch::kFloat32));
        a.lse = out.lse.data_ptr<float>();
    }

    a.cu_seq_k = cu_seq_k.data_ptr<int32_t>();
    a.max_seq_k = max_seq_k;
    a.total_k = block_table ? 0u : (uint32_t)std::min<int64_t>(total_k, 0xFFFFFFFFll);  // a packed cache's rows are the batch's keys
    a.batch = batch;
    a.head_q = head_q;
    a.head_k = head_k;
    a.dim = dim;
    a.dim_v = dim_v;
    a.softmax_scale = softmax_scale.has_value() ? (float)softmax_scale.value() : 0.0f;
    a.stream = stream;
    if (fp8_cache) {
        TORCH_CHECK(v_.has_value(), "a quantised cache needs a value tensor");
        a.kv_dtype = int8_cache ? DA_KV_INT8 : DA_KV_FP8_E4M3;
        a.k_scale = (float)k_scale;
        a.v_scale = (float)v_scale;
    }
    if (block_table) {
        TORCH_CHECK(block_table->dtype() == torch::kInt32, "block_table must have dtype int32");
        TORCH_CHECK(block_table->is_cuda() && block_table->device() == q.device(), "all tensors must be on one device");
        TORCH_CHECK(block_table->dim() == 2 && block_table->size(0) == batch && block_table->stride(1) == 1,
                    "block_table must be [batch, blocks] with a contiguous last dimension");
        a.block_table = block_table->data_ptr<int32_t>();
        a.block_table_stride = block_table->stride(0);
        a.page_size = (int32_t)page_size;
    }

    // Split partials come from torch's caching allocator, which is ordered on the current stream: calls
    // on different streams of one device never share scratch, and nothing is allocated from the driver
    // once the allocator has warmed up (so the call can be captured in a CUDA graph).
    at::Tensor workspace;
    const size_t ws_bytes = da_decode_workspace_bytes(&a);
    if (ws_bytes > 0) {
        workspace = torch::empty({(int64_t)ws_bytes}, q.options().dtype(torch::kUInt8));
        a.workspace = workspace.data_ptr();
        a.workspace_bytes = ws_bytes;
    }
    const int rc = da_decode_fwd(&a);
    TORCH_CHECK(rc == DA_OK, "decoding_attn: ", da_status_string(rc), ": ", da_last_error());
    return out;
}

// Reference signature (decoding_torch.cpp:19-21).
at::Tensor fwd(const at::Tensor &q, const at::Tensor &k, std::optional<at::Tensor> v_, std::optional<at::Tensor> o_,
               const at::Tensor &cu_seq_k, const int64_t max_seq_k, const int64_t dim_v, const bool is_alibi) {
    return run(q, k, v_, o_, cu_seq_k, max_seq_k, dim_v, is_alibi, std::nullopt, false).o;
}

pybind11::object dmha_fwd(const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const at::Tensor &cu_seq_k,
                          int64_t max_seq_k, bool is_alibi, std::optional<double> softmax_scale,
                          std::optional<at::Tensor> out, bool return_lse, double k_scale, double v_scale) {
    TORCH_CHECK(v.dim() == 3, "value must be 3-D");
    Outputs r = run(q, k, v, out, cu_seq_k, max_seq_k, v.size(2), is_alibi, softmax_scale, return_lse, nullptr, 0,
                    k_scale, v_scale);
    if (return_lse) return pybind11::cast(std::make_tuple(r.o, r.lse));
    return pybind11::cast(r.o);
}

pybind11::object dmla_fwd(const at::Tensor &q, const at::Tensor &kv, const at::Tensor &cu_seq_k, int64_t max_seq_k,
                          int64_t dim_v, bool is_alibi, std::optional<double> softmax_scale,
                          std::optional<at::Tensor> out, bool return_lse) {
    // The reference's fwd() keeps is_alibi when v_ is None (csrc/torch/decoding_torch.cpp:19-21, :76-77).
    Outputs r = run(q, kv, std::nullopt, out, cu_seq_k, max_seq_k, dim_v, is_alibi, softmax_scale, return_lse);
    if (return_lse) return pybind11::cast(std::make_tuple(r.o, r.lse));
    return pybind11::cast(r.o);
}

// Paged cache: k_cache [num_pages, page_size, head_k, dim], v_cache the same with dim_v (or None for the
// latent-KV shape), block_table int32 [batch, blocks].  No counterpart in the reference's binding; its
// Python benchmark builds these layouts for the libraries it compares against
// (benchmarks/python/benchmark_decoding_attn.py:129-151, :182-190).
pybind11::object paged_fwd(const at::Tensor &q, const at::Tensor &k_cache, std::optional<at::Tensor> v_cache,
                           const at::Tensor &cu_seq_k, const at::Tensor &block_table, int64_t max_seq_k, int64_t dim_v,
                           bool is_alibi, std::optional<double> softmax_scale, std::optional<at::Tensor> out,
                           bool return_lse) {
    TORCH_CHECK(k_cache.dim() == 4 && k_cache.is_contiguous(), "k_cache must be a contiguous [pages, page_size, head_k, dim]");
    const int64_t page_size = k_cache.size(1);
    const at::Tensor k = k_cache.view({-1, k_cache.size(2), k_cache.size(3)});
    std::optional<at::Tensor> v;
    if (v_cache.has_value()) {
        TORCH_CHECK(v_cache->dim() == 4 && v_cache->is_contiguous() && v_cache->size(0) == k_cache.size(0) &&
                        v_cache->size(1) == page_size,
                    "v_cache must be a contiguous [pages, page_size, head_k, dim_v] like k_cache");
        v = v_cache->view({-1, v_cache->size(2), v_cache->size(3)});
    }
    Outputs r = run(q, k, v, out, cu_seq_k, max_seq_k, dim_v, is_alibi, softmax_scale, return_lse, &block_table, page_size);
    if (return_lse) return pybind11::cast(std::make_tuple(r.o, r.lse));
    return pybind11::cast(r.o);
}

// part_o fp32 [parts, rows..., dim_v], part_lse fp32 [parts, rows...] -> (o [rows..., dim_v], lse).
std::tuple<at::Tensor, at::Tensor> merge_partials(const at::Tensor &part_o, const at::Tensor &part_lse,
                                                  at::ScalarType out_dtype) {
    DA_CHECK_DEVICE(part_o);
    DA_CHECK_DEVICE(part_lse);
    DA_CHECK_CONTIGUOUS(part_o);
    DA_CHECK_CONTIGUOUS(part_lse);
    TORCH_CHECK(part_o.dtype() == torch::kFloat32 && part_lse.dtype() == torch::kFloat32, "partials must be fp32");
    TORCH_CHECK(out_dtype == torch::kFloat16 || out_dtype == torch::kBFloat16, "output must be fp16 or bf16");
    TORCH_CHECK(part_o.dim() >= 2 && part_lse.dim() == part_o.dim() - 1, "part_o [parts, ..., dim_v], part_lse [parts, ...]");
    const int64_t parts = part_o.size(0), dim_v = part_o.size(-1);
    const int64_t rows = part_lse.numel() / parts;
    TORCH_CHECK(part_o.numel() == parts * rows * dim_v, "part_o / part_lse shapes disagree");
    const at::cuda::CUDAGuard guard(part_o.device());
    auto out_shape = part_o.sizes().vec();
    out_shape.erase(out_shape.begin());
    at::Tensor o = torch::empty(out_shape, part_o.options().dtype(out_dtype));
    auto lse_shape = part_lse.sizes().vec();
    lse_shape.erase(lse_shape.begin());
    at::Tensor lse = torch::empty(lse_shape, part_lse.options());
    const int rc = da_merge_partials(part_o.data_ptr<float>(), part_lse.data_ptr<float>(), (int32_t)parts, rows,
                                     (int32_t)dim_v, rows * dim_v, dim_v, rows, 1, o.data_ptr(), nullptr,
                                     lse.data_ptr<float>(), out_dtype == torch::kBFloat16,
                                     at::cuda::getCurrentCUDAStream().stream());
    TORCH_CHECK(rc == DA_OK, "decoding_attn: ", da_status_string(rc), ": ", da_last_error());
    return {o, lse};
}

// ---- caches of 8- and 4-bit codes with a scale per (token, KV head) ----------------------------
struct QuantCache {
    int32_t kv_dtype;
    int64_t rows, head_k, dim, page_size;  // page_size 0: packed [rows, head_k, dim]
};

QuantCache check_cache(const at::Tensor &k, const at::Tensor &v, const at::Tensor &k_scale, const at::Tensor &v_scale,
                       const at::Device &device) {
    QuantCache c;
    switch (k.scalar_type()) {
        case at::kFloat8_e4m3fn: c.kv_dtype = DA_KV_FP8_E4M3; break;
        case at::kChar: c.kv_dtype = DA_KV_INT8; break;
        case at::kByte: c.kv_dtype = DA_KV_INT4; break;
        default: TORCH_CHECK(false, "k_cache must have dtype float8_e4m3fn, int8 or uint8 (two int4 codes a byte)");
    }
    TORCH_CHECK(v.dtype() == k.dtype(), "key and value caches must have the same dtype");
    TORCH_CHECK(k_scale.dtype() == torch::kFloat32 && v_scale.dtype() == torch::kFloat32, "scales must have dtype float32");
    for (const at::Tensor *t : {&k, &v, &k_scale, &v_scale}) {
        TORCH_CHECK(t->is_cuda() && t->device() == device, "all tensors must be on one CUDA device");
        TORCH_CHECK(t->is_contiguous(), "caches and scales must be contiguous");
    }
    TORCH_CHECK(k.dim() == 3 || k.dim() == 4, "k_cache must be [rows, head_k, dim] or [pages, page_size, head_k, dim]");
    TORCH_CHECK(v.sizes() == k.sizes(), "k_cache and v_cache must have the same shape");
    TORCH_CHECK(k_scale.sizes() == k.sizes().slice(0, k.dim() - 1) && v_scale.sizes() == k_scale.sizes(),
                "scales must have the caches' shape without the last dimension");
    c.page_size = k.dim() == 4 ? k.size(1) : 0;
    c.rows = k.dim() == 4 ? k.size(0) * k.size(1) : k.size(0);
    c.head_k = k.size(-2);
    c.dim = k.size(-1) * (c.kv_dtype == DA_KV_INT4 ? 2 : 1);
    return c;
}

// Rows that do not overlap, with their elements side by side: a copy, if they are not like that.
at::Tensor dense(const at::Tensor &x) { return x.dim() == 0 || (x.stride(-1) == 1 && !rows_overlap(x)) ? x : x.contiguous(); }
std::optional<at::Tensor> dense(const std::optional<at::Tensor> &x) {
    return x.has_value() ? std::optional<at::Tensor>(dense(*x)) : std::nullopt;
}

void check_rows(const at::Tensor &x, const char *name, int64_t tokens, const QuantCache &c, const at::Device &device) {
    TORCH_CHECK(x.is_cuda() && x.device() == device, "all tensors must be on one CUDA device");
    TORCH_CHECK(x.dim() == 3 && x.size(0) == tokens && x.size(1) == c.head_k && x.size(2) == c.dim, name,
                " must have shape (tokens, head_k, dim) with the caches' head_k and dim");
    TORCH_CHECK(x.stride(2) == 1 && (c.head_k == 1 || x.stride(1) == c.dim), "heads must be contiguous inside a token row");
    TORCH_CHECK(!rows_overlap(x), name, " must have rows of its own for every token");
}

const int64_t *check_slots(const std::optional<at::Tensor> &slots, int64_t tokens, const at::Device &device) {
    if (!slots.has_value()) return nullptr;
    TORCH_CHECK(slots->is_cuda() && slots->device() == device, "all tensors must be on one CUDA device");
    TORCH_CHECK(slots->dtype() == torch::kInt64 && slots->dim() == 1 && slots->size(0) == tokens && slots->is_contiguous(),
                "slots must be a contiguous int64 tensor with one element per token");
    return slots->data_ptr<int64_t>();
}

da_kv_rows_args_t rows_args(const at::Tensor &k, const at::Tensor &v, const at::Tensor &k_cache, const at::Tensor &v_cache,
                            const at::Tensor &k_scale, const at::Tensor &v_scale, const QuantCache &c) {
    da_kv_rows_args_t a;
    std::memset(&a, 0, sizeof(a));
    a.struct_size = sizeof(a);
    a.kv_dtype = c.kv_dtype;
    a.x_dtype = k.scalar_type() == at::kHalf ? DA_ROWS_FP16 : (k.scalar_type() == at::kBFloat16 ? DA_ROWS_BF16 : DA_ROWS_FP32);
    a.k = k.data_ptr();
    a.v = v.data_ptr();
    a.k_cache = k_cache.data_ptr();
    a.v_cache = v_cache.data_ptr();
    a.k_scale = k_scale.data_ptr<float>();
    a.v_scale = v_scale.data_ptr<float>();
    a.tokens = k.size(0);
    a.cache_rows = c.rows;
    a.head_k = c.head_k;
    a.dim = c.dim;
    // (a tensor of one token may carry any stride; the library wants one that covers the row)
    a.k_row_stride = a.tokens > 1 ? k.stride(0) : 0;
    a.v_row_stride = a.tokens > 1 ? v.stride(0) : 0;
    a.stream = at::cuda::getCurrentCUDAStream().stream();
    return a;
}

void kv_cache_write(const at::Tensor &k_, const at::Tensor &v_, const at::Tensor &k_cache, const at::Tensor &v_cache,
                    const at::Tensor &k_scale, const at::Tensor &v_scale, std::optional<at::Tensor> slots) {
    const at::Tensor k = dense(k_), v = dense(v_);
    TORCH_CHECK(k.dtype() == torch::kFloat16 || k.dtype() == torch::kBFloat16,
                "Decoding-Attention only support FP16 and BF16 data type");
    TORCH_CHECK(v.dtype() == k.dtype(), "key and value must have the same dtype");
    const QuantCache c = check_cache(k_cache, v_cache, k_scale, v_scale, k.device());
    TORCH_CHECK(k.dim() == 3, "key and value must be 3-D");
    check_rows(k, "key", k.size(0), c, k.device());
    check_rows(v, "value", k.size(0), c, k.device());
    const at::cuda::CUDAGuard guard(k.device());
    da_kv_rows_args_t a = rows_args(k, v, k_cache, v_cache, k_scale, v_scale, c);
    a.slots = check_slots(slots, a.tokens, k.device());
    const int rc = da_kv_cache_write(&a);
    TORCH_CHECK(rc == DA_OK, "decoding_attn: ", da_status_string(rc), ": ", da_last_error());
}

std::tuple<at::Tensor, at::Tensor> kv_cache_read(const at::Tensor &k_cache, const at::Tensor &v_cache,
                                                 const at::Tensor &k_scale, const at::Tensor &v_scale,
                                                 std::optional<at::Tensor> slots, at::ScalarType dtype,
                                                 std::optional<std::tuple<at::Tensor, at::Tensor>> out) {
    const at::Device device = k_cache.device();
    const QuantCache c = check_cache(k_cache, v_cache, k_scale, v_scale, device);
    TORCH_CHECK(dtype == at::kHalf || dtype == at::kBFloat16 || dtype == at::kFloat, "dtype must be float16, bfloat16 or float32");
    const int64_t tokens = slots.has_value() ? slots->numel() : c.rows;
    const at::cuda::CUDAGuard guard(device);
    at::Tensor k, v;
    if (out.has_value()) {
        k = std::get<0>(*out);
        v = std::get<1>(*out);
        TORCH_CHECK(k.scalar_type() == dtype && v.scalar_type() == dtype, "Output must have the dtype asked for");
        check_rows(k, "out[0]", tokens, c, device);
        check_rows(v, "out[1]", tokens, c, device);
    } else {
        // (all of it is written, and the call is short: straight to the allocator)
        const std::array<int64_t, 3> shape = {tokens, c.head_k, c.dim};
        k = at::detail::empty_cuda(shape, dtype, device, std::nullopt);
        v = at::detail::empty_cuda(shape, dtype, device, std::nullopt);
    }
    da_kv_rows_args_t a = rows_args(k, v, k_cache, v_cache, k_scale, v_scale, c);
    a.slots = check_slots(slots, tokens, device);
    const int rc = da_kv_cache_read(&a);
    TORCH_CHECK(rc == DA_OK, "decoding_attn: ", da_status_string(rc), ": ", da_last_error());
    return {k, v};
}

// q and the outputs of the decode calls below.
void check_query(const at::Tensor &q, int64_t batch, int64_t head_k, int64_t dim) {
    TORCH_CHECK(q.dtype() == torch::kFloat16 || q.dtype() == torch::kBFloat16,
                "Decoding-Attention only support FP16 and BF16 data type");
    DA_CHECK_DEVICE(q);
    TORCH_CHECK(q.dim() == 3, "query must be 3-D");
    TORCH_CHECK(batch > 0, "batch size must be positive");
    TORCH_CHECK(q.size(0) == batch, "one query token per sequence: q.size(0) must equal cu_seq_k.numel() - 1");
    TORCH_CHECK(q.size(2) == dim, "query and key must have the same head dim");
    TORCH_CHECK(head_k > 0 && q.size(1) % head_k == 0, "number of heads in key/value must divide number of heads in query");
    TORCH_CHECK(q.stride(2) == 1 && (q.size(1) == 1 || q.stride(1) == dim), "heads must be contiguous inside a token row");
}
Outputs make_outputs(const at::Tensor &q, const std::optional<at::Tensor> &out, bool want_lse) {
    Outputs r;
    if (out.has_value()) {
        r.o = out.value();
        TORCH_CHECK(r.o.dtype() == q.dtype(), "Output must have the same dtype as inputs");
        TORCH_CHECK(r.o.is_cuda() && r.o.device() == q.device(), "all tensors must be on one device");
        TORCH_CHECK(r.o.sizes() == q.sizes(), "out must have the shape of the query");
        TORCH_CHECK(r.o.stride(2) == 1 && (q.size(1) == 1 || r.o.stride(1) == q.size(2)), "heads must be contiguous inside a token row");
        TORCH_CHECK(!rows_overlap(r.o), "out must have rows of its own for every sequence");
    } else {
        r.o = torch::empty(q.sizes(), q.options());
    }
    if (want_lse) r.lse = torch::empty({q.size(0), q.size(1)}, q.options().dtype(torch::kFloat32));
    return r;
}
void check_cu(const at::Tensor &cu_seq_k, const at::Device &device) {
    TORCH_CHECK(cu_seq_k.dtype() == torch::kInt32, "cu_seq_k must have dtype int32");
    TORCH_CHECK(cu_seq_k.is_cuda() && cu_seq_k.device() == device, "all tensors must be on one device");
    TORCH_CHECK(cu_seq_k.dim() == 1 && cu_seq_k.is_contiguous(), "cu_seq_k must be a contiguous 1-D tensor");
}
void check_table(const at::Tensor &table, int64_t batch, const at::Device &device) {
    TORCH_CHECK(table.dtype() == torch::kInt32, "block_table must have dtype int32");
    TORCH_CHECK(table.is_cuda() && table.device() == device, "all tensors must be on one device");
    TORCH_CHECK(table.dim() == 2 && table.size(0) == batch && table.size(1) > 0 && (table.size(1) == 1 || table.stride(1) == 1),
                "block_table must be [batch, blocks] with a contiguous last dimension");
}
int64_t row_stride(const at::Tensor &x) { return x.size(0) > 1 ? x.stride(0) : 0; }

pybind11::object quantized_fwd(const at::Tensor &q_, const at::Tensor &k_cache, const at::Tensor &v_cache,
                               const at::Tensor &k_scale, const at::Tensor &v_scale, const at::Tensor &cu_seq_k,
                               bool is_alibi, std::optional<double> softmax_scale, std::optional<at::Tensor> out,
                               bool return_lse, std::optional<at::Tensor> block_table) {
    const at::Tensor q = dense(q_);
    const QuantCache c = check_cache(k_cache, v_cache, k_scale, v_scale, q.device());
    check_cu(cu_seq_k, q.device());
    const int64_t batch = cu_seq_k.numel() - 1;
    check_query(q, batch, c.head_k, c.dim);
    TORCH_CHECK(block_table.has_value() == (c.page_size > 0), "a paged cache (4-D) needs a block_table, a packed one takes none");
    const at::cuda::CUDAGuard guard(q.device());
    const Outputs r = make_outputs(q, out, return_lse);
    da_quant_decode_args_t a;
    std::memset(&a, 0, sizeof(a));
    a.struct_size = sizeof(a);
    a.is_bf16 = q.scalar_type() == at::kBFloat16;
    a.is_alibi = is_alibi;
    a.kv_dtype = c.kv_dtype;
    a.q = q.data_ptr();
    a.k = k_cache.data_ptr();
    a.v = v_cache.data_ptr();
    a.k_scale = k_scale.data_ptr<float>();
    a.v_scale = v_scale.data_ptr<float>();
    a.o = r.o.data_ptr();
    a.lse = return_lse ? r.lse.data_ptr<float>() : nullptr;
    a.cu_seq_k = cu_seq_k.data_ptr<int32_t>();
    a.rows = c.rows;
    a.batch = batch;
    a.head_q = q.size(1);
    a.head_k = c.head_k;
    a.dim = c.dim;
    a.q_row_stride = row_stride(q);
    a.o_row_stride = row_stride(r.o);
    if (block_table.has_value()) {
        check_table(*block_table, batch, q.device());
        a.block_table = block_table->data_ptr<int32_t>();
        a.block_table_stride = batch > 1 ? block_table->stride(0) : block_table->size(1);
        a.table_blocks = block_table->size(1);
        a.page_size = (int32_t)c.page_size;
    }
    a.softmax_scale = softmax_scale.has_value() ? (float)softmax_scale.value() : 0.0f;
    a.stream = at::cuda::getCurrentCUDAStream().stream();
    const size_t bytes = da_quant_decode_workspace_bytes(&a);
    at::Tensor workspace;
    if (bytes > 0) {
        workspace = torch::empty({(int64_t)bytes}, q.options().dtype(torch::kUInt8));
        a.workspace = workspace.data_ptr();
        a.workspace_bytes = bytes;
    }
    const int rc = da_quant_decode_fwd(&a);
    TORCH_CHECK(rc == DA_OK, "decoding_attn: ", da_status_string(rc), ": ", da_last_error());
    if (return_lse) return pybind11::cast(std::make_tuple(r.o, r.lse));
    return pybind11::cast(r.o);
}

pybind11::object shared_prefix_fwd(const at::Tensor &q_, const std::optional<at::Tensor> &prefix_k,
                                   const std::optional<at::Tensor> &prefix_v, const at::Tensor &own_k, const at::Tensor &own_v,
                                   const at::Tensor &cu_seq_k, bool is_alibi, std::optional<double> softmax_scale,
                                   std::optional<at::Tensor> out, bool return_lse, const std::optional<at::Tensor> &k_scale,
                                   const std::optional<at::Tensor> &v_scale, const std::optional<at::Tensor> &block_table,
                                   const std::optional<at::Tensor> &prefix_table, std::optional<int64_t> prefix_len) {
    const at::Tensor q = dense(q_);
    const std::optional<at::Tensor> k_prefix_ = dense(prefix_k), v_prefix_ = dense(prefix_v);
    const at::Tensor k = k_scale.has_value() ? own_k : dense(own_k), v = k_scale.has_value() ? own_v : dense(own_v);
    const at::Device device = q.device();
    TORCH_CHECK(k_scale.has_value() == v_scale.has_value(), "k_scale and v_scale come together");
    TORCH_CHECK(k_prefix_.has_value() == v_prefix_.has_value(), "k_prefix and v_prefix come together");
    check_cu(cu_seq_k, device);
    const int64_t batch = cu_seq_k.numel() - 1;
    da_prefix_decode_args_t a;
    std::memset(&a, 0, sizeof(a));
    a.struct_size = sizeof(a);

    // the sequences' own keys: codes with scales, or rows of q's type, packed or in pages
    int64_t page_size = 0;
    if (k_scale.has_value()) {
        const QuantCache c = check_cache(k, v, *k_scale, *v_scale, device);
        a.kv_dtype = c.kv_dtype;
        a.k_scale = k_scale->data_ptr<float>();
        a.v_scale = v_scale->data_ptr<float>();
        a.rows = c.rows;
        a.head_k = c.head_k;
        a.dim = c.dim;
        page_size = c.page_size;
    } else {
        TORCH_CHECK(k.dtype() == q.dtype() && v.dtype() == q.dtype(), "query, key and value must have the same dtype");
        TORCH_CHECK(k.is_cuda() && k.device() == device && v.is_cuda() && v.device() == device, "all tensors must be on one device");
        TORCH_CHECK(k.dim() == 3 || k.dim() == 4, "key must be [total_k, head_k, dim] or [pages, page_size, head_k, dim]");
        TORCH_CHECK(v.sizes() == k.sizes(), "key and value must have the same shape");
        a.head_k = k.size(-2);
        a.dim = k.size(-1);
        if (k.dim() == 4) {
            TORCH_CHECK(k.is_contiguous() && v.is_contiguous(), "a paged cache must be contiguous");
            page_size = k.size(1);
            a.rows = k.size(0) * page_size;
        } else {
            a.rows = k.size(0);
            for (const at::Tensor *t : {&k, &v})
                TORCH_CHECK(t->stride(2) == 1 && (a.head_k == 1 || t->stride(1) == a.dim), "heads must be contiguous inside a token row");
            a.k_row_stride = row_stride(k);
            a.v_row_stride = row_stride(v);
        }
    }
    check_query(q, batch, a.head_k, a.dim);
    TORCH_CHECK(block_table.has_value() == (page_size > 0), "a paged cache (4-D) needs a block_table, a packed one takes none");

    // the prefix: rows of its own, or pages of a pool of its own or of the sequences'
    TORCH_CHECK(k_prefix_.has_value() || prefix_table.has_value(), "k_prefix and v_prefix, or a prefix_table into k and v, must be given");
    TORCH_CHECK(k_prefix_.has_value() || (page_size > 0 && !k_scale.has_value()), "a prefix in the sequences' own cache needs a paged cache in q's dtype");
    const at::Tensor &kp = k_prefix_.has_value() ? *k_prefix_ : k;
    const at::Tensor &vp = v_prefix_.has_value() ? *v_prefix_ : v;
    TORCH_CHECK(kp.is_cuda() && kp.device() == device && vp.is_cuda() && vp.device() == device, "all tensors must be on one device");
    TORCH_CHECK(kp.dtype() == q.dtype() && vp.dtype() == q.dtype(), "the prefix must have the dtype of the query");
    TORCH_CHECK(kp.dim() == (prefix_table.has_value() ? 4 : 3), "the prefix must be [prefix_len, head_k, dim], or [pages, page_size, head_k, dim] with a prefix_table");
    TORCH_CHECK(vp.sizes() == kp.sizes() && kp.size(-2) == a.head_k && kp.size(-1) == a.dim, "prefix and own keys must have the same head_k and dim");
    if (prefix_table.has_value()) {
        TORCH_CHECK(kp.is_contiguous() && vp.is_contiguous(), "a paged prefix must be contiguous");
        TORCH_CHECK(prefix_table->dtype() == torch::kInt32 && prefix_table->dim() == 1 && prefix_table->is_contiguous(), "prefix_table must be a contiguous 1-D int32 tensor");
        TORCH_CHECK(prefix_table->is_cuda() && prefix_table->device() == device, "all tensors must be on one device");
        TORCH_CHECK(prefix_len.has_value(), "a paged prefix needs prefix_len");
        a.prefix_len = *prefix_len;
        a.prefix_page_size = (int32_t)kp.size(1);
        a.prefix_rows = kp.size(0) * kp.size(1);
        a.prefix_table = prefix_table->data_ptr<int32_t>();
        TORCH_CHECK(a.prefix_len <= prefix_table->numel() * kp.size(1), "prefix_len exceeds the pages of prefix_table");
    } else {
        for (const at::Tensor *t : {&kp, &vp})
            TORCH_CHECK(t->stride(2) == 1 && (a.head_k == 1 || t->stride(1) == a.dim), "heads must be contiguous inside a token row");
        a.prefix_len = prefix_len.has_value() ? *prefix_len : kp.size(0);
        a.prefix_rows = kp.size(0);
        a.k_prefix_row_stride = row_stride(kp);
        a.v_prefix_row_stride = row_stride(vp);
    }

    const at::cuda::CUDAGuard guard(device);
    const Outputs r = make_outputs(q, out, return_lse);
    a.is_bf16 = q.scalar_type() == at::kBFloat16;
    a.is_alibi = is_alibi;
    a.q = q.data_ptr();
    a.k_prefix = kp.data_ptr();
    a.v_prefix = vp.data_ptr();
    a.k = k.data_ptr();
    a.v = v.data_ptr();
    a.o = r.o.data_ptr();
    a.lse = return_lse ? r.lse.data_ptr<float>() : nullptr;
    a.cu_seq_k = cu_seq_k.data_ptr<int32_t>();
    a.batch = batch;
    a.head_q = q.size(1);
    a.q_row_stride = row_stride(q);
    a.o_row_stride = row_stride(r.o);
    if (block_table.has_value()) {
        check_table(*block_table, batch, device);
        a.block_table = block_table->data_ptr<int32_t>();
        a.block_table_stride = batch > 1 ? block_table->stride(0) : block_table->size(1);
        a.table_blocks = block_table->size(1);
        a.page_size = (int32_t)page_size;
    }
    a.softmax_scale = softmax_scale.has_value() ? (float)softmax_scale.value() : 0.0f;
    a.stream = at::cuda::getCurrentCUDAStream().stream();
    const size_t bytes = da_prefix_decode_workspace_bytes(&a);
    at::Tensor workspace;
    if (bytes > 0) {
        workspace = torch::empty({(int64_t)bytes}, q.options().dtype(torch::kUInt8));
        a.workspace = workspace.data_ptr();
        a.workspace_bytes = bytes;
    }
    const int rc = da_prefix_decode_fwd(&a);
    TORCH_CHECK(rc == DA_OK, "decoding_attn: ", da_status_string(rc), ": ", da_last_error());
    if (return_lse) return pybind11::cast(std::make_tuple(r.o, r.lse));
    return pybind11::cast(r.o);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    namespace py = pybind11;
    m.doc() = "Decoding-Attention (B200)";
    m.def("fwd", &fwd, "Forward pass", py::arg("q"), py::arg("k"), py::arg("v_"), py::arg("o_"), py::arg("cu_seq_k"),
          py::arg("max_seq_k"), py::arg("dim_v"), py::arg("is_alibi"));
    m.def("dmha_fwd", &dmha_fwd, "MHA/GQA/MQA decode", py::arg("q"), py::arg("k"), py::arg("v"), py::arg("cu_seq_k"),
          py::arg("max_seq_k"), py::arg("is_alibi") = false, py::arg("softmax_scale") = py::none(),
          py::arg("out") = py::none(), py::arg("return_lse") = false, py::arg("k_scale") = 1.0, py::arg("v_scale") = 1.0);
    m.def("dmla_fwd", &dmla_fwd, "MLA decode (latent KV)", py::arg("q"), py::arg("kv"), py::arg("cu_seq_k"),
          py::arg("max_seq_k"), py::arg("dim_v") = 512, py::arg("is_alibi") = false,
          py::arg("softmax_scale") = py::none(), py::arg("out") = py::none(), py::arg("return_lse") = false);
    m.def("paged_fwd", &paged_fwd, "Decode over a paged KV cache", py::arg("q"), py::arg("k_cache"), py::arg("v_cache"),
          py::arg("cu_seq_k"), py::arg("block_table"), py::arg("max_seq_k"), py::arg("dim_v"), py::arg("is_alibi") = false,
          py::arg("softmax_scale") = py::none(), py::arg("out") = py::none(), py::arg("return_lse") = false);
    m.def("merge_partials", &merge_partials, "LSE merge of key-range partials", py::arg("part_o"),
          py::arg("part_lse"), py::arg("out_dtype"));
    m.def("kv_cache_write", &kv_cache_write, "Quantise K and V rows into a cache", py::arg("k"), py::arg("v"),
          py::arg("k_cache"), py::arg("v_cache"), py::arg("k_scale"), py::arg("v_scale"), py::arg("slots") = py::none());
    m.def("kv_cache_read", &kv_cache_read, "Rows of a quantised cache", py::arg("k_cache"), py::arg("v_cache"),
          py::arg("k_scale"), py::arg("v_scale"), py::arg("slots"), py::arg("dtype"), py::arg("out") = py::none());
    m.def("quantized_fwd", &quantized_fwd, "Decode over a cache with a scale per token and head", py::arg("q"),
          py::arg("k_cache"), py::arg("v_cache"), py::arg("k_scale"), py::arg("v_scale"), py::arg("cu_seq_k"),
          py::arg("is_alibi") = false, py::arg("softmax_scale") = py::none(), py::arg("out") = py::none(),
          py::arg("return_lse") = false, py::arg("block_table") = py::none());
    m.def("shared_prefix_fwd", &shared_prefix_fwd, "Decode behind a prefix that the batch shares", py::arg("q"),
          py::arg("k_prefix"), py::arg("v_prefix"), py::arg("k"), py::arg("v"), py::arg("cu_seq_k"),
          py::arg("is_alibi") = false, py::arg("softmax_scale") = py::none(), py::arg("out") = py::none(),
          py::arg("return_lse") = false, py::arg("k_scale") = py::none(), py::arg("v_scale") = py::none(),
          py::arg("block_table") = py::none(), py::arg("prefix_table") = py::none(), py::arg("prefix_len") = py::none());
    m.def("launch_count", []() { return da_launch_count(); });
    m.def("device_status", []() { return da_device_status(); });
}
