// bindings.cpp -- the torch extension module `long_context_attention_kernels`, a thin
// pybind11 layer over the C ABI in include/lca.h.
//
// Mirrors the reference extension (csrc/bindings.cpp:31-80): same module name, same
// function `sliding_window_attention_forward(Q, K, V, window_size, global_tokens, scale)`
// returning a new fp32 tensor allocated through torch's caching allocator, launched on
// the current CUDA stream, errors raised as RuntimeError (IndexError for an out-of-range
// global token, as the reference's mask construction raises).  Differences: fp16 and
// bf16 inputs, head_dim 64 or 128, and launch/device errors are checked.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>

#include <vector>

#include "lca.h"

namespace {

void check_input(const torch::Tensor& t, const char* name) {
    TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
    TORCH_CHECK(t.scalar_type() == torch::kFloat16 || t.scalar_type() == torch::kBFloat16, name,
                " must be fp16 or bf16");
    TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
}

void raise_status(int st, const char* what) {
    if (st == LCA_OK) return;
    const char* detail = lca_last_error();
    if (st == LCA_ERR_INDEX) TORCH_CHECK_INDEX(false, what, ": ", detail);
    TORCH_CHECK(false, what, " failed (", lca_status_string(st), "): ", detail);
}

std::vector<torch::Tensor> forward_impl(const torch::Tensor& Q, const torch::Tensor& K, const torch::Tensor& V,
                                        int64_t window_size, const std::vector<int64_t>& globals, double scale,
                                        bool want_lse, c10::ScalarType out_type = torch::kFloat32,
                                        bool causal = false, const std::vector<int64_t>& head_windows = {},
                                        int64_t dilation = 1, const std::vector<int64_t>& cu_seqlens = {},
                                        bool token_major = false) {
    check_input(Q, "Q");
    check_input(K, "K");
    check_input(V, "V");
    TORCH_CHECK(Q.dim() == 4, token_major ? "Q must be [batch, seq_len, heads, head_dim]"
                                          : "Q must be [batch, heads, seq_len, head_dim]");
    TORCH_CHECK(K.sizes() == Q.sizes() && V.sizes() == Q.sizes(), "Q, K and V must have the same shape");
    TORCH_CHECK(K.scalar_type() == Q.scalar_type() && V.scalar_type() == Q.scalar_type(),
                "Q, K and V must have the same dtype");
    TORCH_CHECK(K.device() == Q.device() && V.device() == Q.device(), "Q, K and V must be on the same device");
    const int64_t batch = Q.size(0), heads = Q.size(token_major ? 2 : 1), seq_len = Q.size(token_major ? 1 : 2),
                  head_dim = Q.size(3);
    TORCH_CHECK(head_dim == 64 || head_dim == 128, "head_dim must be 64 or 128 (got ", head_dim, ")");
    TORCH_CHECK(window_size >= 0, "window_size must be >= 0 (got ", window_size, ")");
    TORCH_CHECK(head_windows.empty() || (int64_t)head_windows.size() == heads,
                "window_size per head needs one radius per head (got ", head_windows.size(), " for ", heads,
                " heads)");
    TORCH_CHECK(out_type == torch::kFloat32 || out_type == torch::kFloat16 || out_type == torch::kBFloat16,
                "out_dtype must be float32, float16 or bfloat16");

    c10::cuda::CUDAGuard guard(Q.device());
    auto O = torch::empty(Q.sizes(), Q.options().dtype(out_type));  // the input's layout
    torch::Tensor L;
    if (want_lse) L = torch::empty({batch, heads, seq_len}, Q.options().dtype(torch::kFloat32));

    const int dtype = Q.scalar_type() == torch::kBFloat16 ? LCA_DTYPE_BF16 : LCA_DTYPE_F16;
    std::vector<int32_t> norm(globals.size() + 1);
    int64_t G = 0;
    if (cu_seqlens.empty())
        raise_status(lca_normalize_global_tokens(globals.data(), (int64_t)globals.size(), seq_len, norm.data(), &G),
                     "global_tokens");
    size_t ws_bytes = 0;
    int64_t wmax = window_size;
    for (int64_t hw : head_windows) wmax = std::max(wmax, hw);
    TORCH_CHECK(dilation >= 1, "dilation must be >= 1");
    TORCH_CHECK(cu_seqlens.empty() || (batch == 1 && dilation == 1),
                "packed sequences take Q of shape [1, heads, total_len, head_dim] and no dilation");
    const int out_dtype = out_type == torch::kFloat32 ? LCA_DTYPE_F32
                          : (out_type == torch::kBFloat16 ? LCA_DTYPE_BF16 : LCA_DTYPE_F16);
    if (!cu_seqlens.empty()) {
        const int64_t nseq = (int64_t)cu_seqlens.size() - 1;
        G = nseq * (int64_t)globals.size();  // an upper bound on the unique global rows
        raise_status(lca_swa_workspace_size(1, heads, seq_len, head_dim, wmax, G, dtype, &ws_bytes),
                     "workspace size");
    } else if (dilation > 1) {
        raise_status(lca_swa_dilated_workspace_size(batch, heads, seq_len, head_dim, wmax, dilation, G, dtype,
                                                    out_dtype, &ws_bytes),
                     "workspace size");
    } else {
        raise_status(lca_swa_workspace_size(batch, heads, seq_len, head_dim, wmax, G, dtype, &ws_bytes),
                     "workspace size");
    }
    torch::Tensor ws;
    void* ws_ptr = nullptr;
    if (ws_bytes > 0) {
        ws = torch::empty({(int64_t)ws_bytes}, Q.options().dtype(torch::kUInt8));
        ws_ptr = ws.data_ptr();
    }
    cudaStream_t stream = at::cuda::getCurrentCUDAStream();
    const int64_t* hw = head_windows.empty() ? nullptr : head_windows.data();
    const int flags = (causal ? LCA_FLAG_CAUSAL : 0) | (token_major ? LCA_FLAG_TOKEN_MAJOR : 0);
    float* lse_ptr = want_lse ? L.data_ptr<float>() : nullptr;
    void* sp = static_cast<void*>(stream);
    int st;
    if (!cu_seqlens.empty())
        st = lca_swa_forward_varlen(Q.data_ptr(), K.data_ptr(), V.data_ptr(), O.data_ptr(), out_dtype, lse_ptr, dtype,
                                    heads, seq_len, head_dim, window_size, hw, static_cast<float>(scale), flags,
                                    cu_seqlens.data(), (int64_t)cu_seqlens.size() - 1, globals.data(),
                                    (int64_t)globals.size(), ws_ptr, ws_bytes, sp);
    else
        st = lca_swa_forward_dilated(Q.data_ptr(), K.data_ptr(), V.data_ptr(), O.data_ptr(), out_dtype, lse_ptr, dtype,
                                     batch, heads, seq_len, head_dim, window_size, hw, dilation,
                                     static_cast<float>(scale), flags, globals.data(), (int64_t)globals.size(), ws_ptr,
                                     ws_bytes, sp);
    raise_status(st, "sliding_window_attention_forward");
    if (want_lse) return {O, L};
    return {O};
}

std::vector<int64_t> tokens_from_tensor(const torch::Tensor& global_tokens) {
    // The reference accepts the index tensor on any device and converts it to int32
    // (csrc/bindings.cpp:47); here it is read on the host (a device tensor costs a copy).
    auto t = global_tokens.to(torch::kCPU, torch::kInt64).contiguous().view({-1});
    const int64_t* p = t.data_ptr<int64_t>();
    return std::vector<int64_t>(p, p + t.numel());
}

torch::Tensor sliding_window_attention_forward(torch::Tensor Q, torch::Tensor K, torch::Tensor V,
                                               int64_t window_size, torch::Tensor global_tokens, double scale) {
    return forward_impl(Q, K, V, window_size, tokens_from_tensor(global_tokens), scale, false)[0];
}

torch::Tensor sliding_window_attention_forward_list(torch::Tensor Q, torch::Tensor K, torch::Tensor V,
                                                    int64_t window_size, std::vector<int64_t> global_tokens,
                                                    double scale) {
    return forward_impl(Q, K, V, window_size, global_tokens, scale, false)[0];
}

std::vector<torch::Tensor> sliding_window_attention_forward_lse(torch::Tensor Q, torch::Tensor K, torch::Tensor V,
                                                                int64_t window_size,
                                                                std::vector<int64_t> global_tokens, double scale) {
    return forward_impl(Q, K, V, window_size, global_tokens, scale, true);
}

std::vector<torch::Tensor> sliding_window_attention_forward_ex(torch::Tensor Q, torch::Tensor K, torch::Tensor V,
                                                               int64_t window_size, std::vector<int64_t> global_tokens,
                                                               double scale, c10::ScalarType out_dtype, bool causal,
                                                               bool want_lse, std::vector<int64_t> head_windows,
                                                               int64_t dilation, std::vector<int64_t> cu_seqlens,
                                                               bool token_major) {
    return forward_impl(Q, K, V, window_size, global_tokens, scale, want_lse, out_dtype, causal, head_windows,
                        dilation, cu_seqlens, token_major);
}

// Gradients of the forward (include/lca.h lca_swa_backward): dQ, dK, dV in fp32, from the
// forward's fp32 O and LSE and the fp32 gradient dO of O.  No counterpart in the reference.
std::vector<torch::Tensor> sliding_window_attention_backward(torch::Tensor Q, torch::Tensor K, torch::Tensor V,
                                                             torch::Tensor O, torch::Tensor LSE, torch::Tensor dO,
                                                             int64_t window_size,
                                                             std::vector<int64_t> global_tokens, double scale) {
    check_input(Q, "Q");
    check_input(K, "K");
    check_input(V, "V");
    TORCH_CHECK(Q.dim() == 4, "Q must be [batch, heads, seq_len, head_dim]");
    TORCH_CHECK(K.sizes() == Q.sizes() && V.sizes() == Q.sizes(), "Q, K and V must have the same shape");
    TORCH_CHECK(K.scalar_type() == Q.scalar_type() && V.scalar_type() == Q.scalar_type(),
                "Q, K and V must have the same dtype");
    for (const torch::Tensor* t : {&O, &dO}) {
        TORCH_CHECK(t->is_cuda() && t->scalar_type() == torch::kFloat32 && t->is_contiguous() &&
                        t->sizes() == Q.sizes(),
                    "O and dO must be contiguous fp32 CUDA tensors of Q's shape");
    }
    const int64_t batch = Q.size(0), heads = Q.size(1), seq_len = Q.size(2), head_dim = Q.size(3);
    TORCH_CHECK(LSE.is_cuda() && LSE.scalar_type() == torch::kFloat32 && LSE.is_contiguous() &&
                    LSE.numel() == batch * heads * seq_len,
                "LSE must be a contiguous fp32 CUDA tensor [batch, heads, seq_len]");
    TORCH_CHECK(head_dim == 64 || head_dim == 128, "head_dim must be 64 or 128 (got ", head_dim, ")");
    TORCH_CHECK(window_size >= 0, "window_size must be >= 0 (got ", window_size, ")");
    c10::cuda::CUDAGuard guard(Q.device());
    const int dtype = Q.scalar_type() == torch::kBFloat16 ? LCA_DTYPE_BF16 : LCA_DTYPE_F16;
    std::vector<int32_t> norm(global_tokens.size() + 1);
    int64_t G = 0;
    raise_status(lca_normalize_global_tokens(global_tokens.data(), (int64_t)global_tokens.size(), seq_len, norm.data(),
                                             &G),
                 "global_tokens");
    size_t ws_bytes = 0;
    raise_status(lca_swa_backward_workspace_size(batch, heads, seq_len, head_dim, window_size, G, dtype, &ws_bytes),
                 "backward workspace size");
    torch::Tensor ws;
    void* ws_ptr = nullptr;
    if (ws_bytes > 0) {
        ws = torch::empty({(int64_t)ws_bytes}, Q.options().dtype(torch::kUInt8));
        ws_ptr = ws.data_ptr();
    }
    auto f32 = Q.options().dtype(torch::kFloat32);
    auto dQ = torch::empty(Q.sizes(), f32), dK = torch::empty(Q.sizes(), f32), dV = torch::empty(Q.sizes(), f32);
    cudaStream_t stream = at::cuda::getCurrentCUDAStream();
    const int st = lca_swa_backward(Q.data_ptr(), K.data_ptr(), V.data_ptr(), O.data_ptr<float>(),
                                    LSE.data_ptr<float>(), dO.data_ptr<float>(), dQ.data_ptr<float>(),
                                    dK.data_ptr<float>(), dV.data_ptr<float>(), dtype, batch, heads, seq_len, head_dim,
                                    window_size, static_cast<float>(scale), global_tokens.data(),
                                    (int64_t)global_tokens.size(), ws_ptr, ws_bytes, static_cast<void*>(stream));
    raise_status(st, "sliding_window_attention_backward");
    return {dQ, dK, dV};
}

int device_error() {
    int code = 0;
    raise_status(lca_device_error(&code), "device_error");
    return code;
}

// ------------------------------------------------------------------ paged 4-bit KV cache
// (include/lca.h lca_kv_* / lca_kv4_* / lca_swa_forward_cached; no counterpart in the reference)

// A new tensor without the dispatcher, which costs a small call a noticeable part of its host time.
torch::Tensor new_tensor(at::IntArrayRef sizes, c10::ScalarType type, const torch::Device& device) {
    return at::detail::empty_cuda(sizes, type, device, c10::nullopt);
}

void check_ints(const torch::Tensor& t, const char* name, int64_t dim, const torch::Device& device) {
    TORCH_CHECK(t.is_cuda() && t.scalar_type() == torch::kInt32 && t.is_contiguous() && t.dim() == dim, name,
                " must be a contiguous int32 CUDA tensor with ", dim, " dimension(s)");
    TORCH_CHECK(t.device() == device, name, " must be on the same device as the others");
}

struct PoolShape {
    int64_t pages, kv_heads, page_size, head_dim;
};

PoolShape check_pool(const torch::Tensor& pool) {
    TORCH_CHECK(pool.is_cuda() && pool.scalar_type() == torch::kUInt8 && pool.is_contiguous() && pool.dim() == 4,
                "pool must be a contiguous uint8 CUDA tensor [pages, kv_heads, page_size, head_dim + 8]");
    return {pool.size(0), pool.size(1), pool.size(2), pool.size(3) - 8};
}

int type_code(c10::ScalarType t, const char* name) {
    TORCH_CHECK(t == torch::kFloat32 || t == torch::kFloat16 || t == torch::kBFloat16, name,
                " must be float32, float16 or bfloat16");
    return t == torch::kFloat32 ? LCA_DTYPE_F32 : (t == torch::kBFloat16 ? LCA_DTYPE_BF16 : LCA_DTYPE_F16);
}

// Elements [from, from + n) of a contiguous 1-D tensor, sharing its storage.  Made directly: eight of
// these through the dispatcher cost more host time than the call they return from.
torch::Tensor part_of(const torch::Tensor& all, int64_t from, int64_t n) {
    auto t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(all.storage()), all.key_set(), all.dtype());
    t.unsafeGetTensorImpl()->set_storage_offset(all.storage_offset() + from);
    t.unsafeGetTensorImpl()->set_sizes_contiguous(c10::IntArrayRef(&n, 1));
    return t;
}

void* current_stream() { return static_cast<void*>(at::cuda::getCurrentCUDAStream().stream()); }

std::vector<torch::Tensor> kv_cache_layout(const torch::Tensor& block_table, const torch::Tensor& seq_lens,
                                           const torch::Tensor& new_lens, const torch::Tensor& free_pages,
                                           const torch::Tensor& free_count, int64_t page_size,
                                           int64_t num_tokens) {
    const auto device = block_table.device();
    check_ints(block_table, "block_table", 2, device);
    check_ints(seq_lens, "seq_lens", 1, device);
    check_ints(new_lens, "new_lens", 1, device);
    check_ints(free_pages, "free_pages", 1, device);
    check_ints(free_count, "free_count", 1, device);
    const int64_t batch = block_table.size(0);
    TORCH_CHECK(seq_lens.size(0) == batch && new_lens.size(0) == batch,
                "seq_lens and new_lens need one length per row of block_table (", batch, ")");
    TORCH_CHECK(free_count.size(0) == 1, "free_count must hold one value");
    TORCH_CHECK(num_tokens >= 0, "num_tokens must be >= 0 (got ", num_tokens, ")");
    c10::cuda::CUDAGuard guard(device);
    const int64_t pad = (num_tokens + 3) / 4 * 4;  // slots and positions on 16-byte boundaries
    auto all = new_tensor({2 * pad + 4 * batch + 2}, torch::kInt32, device);
    int32_t* at = all.data_ptr<int32_t>();
    int32_t *slots = at, *positions = at + pad, *kv_lens = at + 2 * pad, *placed = kv_lens + batch,
            *next = placed + batch, *count = next + batch, *cu = count + 1;
    raise_status(lca_kv_layout(block_table.data_ptr<int32_t>(), batch, block_table.size(1), seq_lens.data_ptr<int32_t>(),
                               new_lens.data_ptr<int32_t>(), free_pages.data_ptr<int32_t>(), free_pages.size(0),
                               free_count.data_ptr<int32_t>(), page_size, num_tokens, slots, positions, cu, kv_lens,
                               placed, next, count, current_stream()),
                 "kv_cache_layout");
    auto part = [&](int32_t* from, int64_t n) { return part_of(all, from - at, n); };
    return {part(slots, num_tokens), part(positions, num_tokens), part(cu, batch + 1), part(kv_lens, batch),
            part(placed, batch),     part(next, batch),           part(count, 1),      part(next, batch + 1)};
}

std::vector<torch::Tensor> kv_cache_release(const torch::Tensor& block_table, const torch::Tensor& seq_lens,
                                            const torch::Tensor& release, const torch::Tensor& free_pages,
                                            const torch::Tensor& free_count, int64_t page_size) {
    const auto device = block_table.device();
    check_ints(block_table, "block_table", 2, device);
    check_ints(seq_lens, "seq_lens", 1, device);
    check_ints(free_pages, "free_pages", 1, device);
    check_ints(free_count, "free_count", 1, device);
    const int64_t batch = block_table.size(0);
    TORCH_CHECK(release.is_cuda() && release.scalar_type() == torch::kBool && release.is_contiguous() &&
                    release.dim() == 1 && release.device() == device,
                "release must be a contiguous bool CUDA tensor with one value per request");
    TORCH_CHECK(seq_lens.size(0) == batch && release.size(0) == batch,
                "seq_lens and release need one value per row of block_table (", batch, ")");
    TORCH_CHECK(free_count.size(0) == 1, "free_count must hold one value");
    c10::cuda::CUDAGuard guard(device);
    auto next = new_tensor({batch + 1}, torch::kInt32, device);
    int32_t* at = next.data_ptr<int32_t>();
    raise_status(lca_kv_release(block_table.data_ptr<int32_t>(), batch, block_table.size(1),
                                seq_lens.data_ptr<int32_t>(), reinterpret_cast<const uint8_t*>(release.data_ptr<bool>()),
                                free_pages.data_ptr<int32_t>(), free_pages.size(0), free_count.data_ptr<int32_t>(),
                                page_size, at, at + batch, current_stream()),
                 "kv_cache_release");
    return {part_of(next, 0, batch), part_of(next, batch, 1), next};
}

void kv_cache_append(const torch::Tensor& pool, const torch::Tensor& k, const torch::Tensor& v, const torch::Tensor& slots) {
    const PoolShape s = check_pool(pool);
    check_ints(slots, "slots", 1, pool.device());
    for (const torch::Tensor* t : {&k, &v}) {
        TORCH_CHECK(t->is_cuda() && t->device() == pool.device() &&
                        (t->scalar_type() == torch::kFloat16 || t->scalar_type() == torch::kBFloat16) &&
                        t->scalar_type() == k.scalar_type(),
                    "k and v must be CUDA tensors of one type, fp16 or bf16, on the pool's device");
        TORCH_CHECK(t->dim() == 3 && t->size(0) == slots.size(0) && t->size(1) == s.kv_heads && t->size(2) == s.head_dim,
                    "k and v must be [tokens, kv_heads, head_dim] = [", slots.size(0), ", ", s.kv_heads, ", ", s.head_dim,
                    "], as the slots and the pool have them");
        TORCH_CHECK(t->size(0) == 0 || t->stride(2) == 1, "the last dimension of k and v must be contiguous");
    }
    c10::cuda::CUDAGuard guard(pool.device());
    raise_status(lca_kv4_append(pool.data_ptr(), s.pages, s.kv_heads, s.page_size, s.head_dim, k.data_ptr(), v.data_ptr(),
                                type_code(k.scalar_type(), "k"), k.stride(0), k.stride(1), v.stride(0), v.stride(1),
                                slots.data_ptr<int32_t>(), slots.size(0), current_stream()),
                 "kv_cache_append");
}

std::vector<torch::Tensor> kv_cache_read(const torch::Tensor& pool, const torch::Tensor& slots, c10::ScalarType out_dtype) {
    const PoolShape s = check_pool(pool);
    check_ints(slots, "slots", 1, pool.device());
    const int code = type_code(out_dtype, "out_dtype");
    c10::cuda::CUDAGuard guard(pool.device());
    auto k = new_tensor({slots.size(0), s.kv_heads, s.head_dim}, out_dtype, pool.device());
    auto v = new_tensor({slots.size(0), s.kv_heads, s.head_dim}, out_dtype, pool.device());
    raise_status(lca_kv4_read(pool.data_ptr(), s.pages, s.kv_heads, s.page_size, s.head_dim, slots.data_ptr<int32_t>(),
                              slots.size(0), k.data_ptr(), v.data_ptr(), code, current_stream()),
                 "kv_cache_read");
    return {k, v};
}

std::vector<torch::Tensor> sliding_window_attention_cached(const torch::Tensor& Q, const torch::Tensor& pool,
                                                           const torch::Tensor& block_table, const torch::Tensor& kv_lens,
                                                           const torch::Tensor& cu_seqlens, int64_t window_size,
                                                           const std::vector<int64_t>& global_tokens, double scale,
                                                           c10::ScalarType out_dtype, bool want_lse,
                                                           const c10::optional<torch::Tensor>& out) {
    const PoolShape s = check_pool(pool);
    const auto device = pool.device();
    check_ints(block_table, "block_table", 2, device);
    check_ints(kv_lens, "kv_lens", 1, device);
    check_ints(cu_seqlens, "cu_seqlens", 1, device);
    const int64_t batch = block_table.size(0);
    TORCH_CHECK(kv_lens.size(0) == batch && cu_seqlens.size(0) == batch + 1,
                "kv_lens needs one length, and cu_seqlens one offset and a last one, per row of block_table (", batch, ")");
    TORCH_CHECK(Q.is_cuda() && Q.device() == device &&
                    (Q.scalar_type() == torch::kFloat16 || Q.scalar_type() == torch::kBFloat16),
                "Q must be an fp16 or bf16 CUDA tensor on the pool's device");
    TORCH_CHECK(Q.dim() == 3 && Q.size(2) == s.head_dim, "Q must be [rows, heads, head_dim] with the pool's head_dim ",
                s.head_dim);
    TORCH_CHECK(Q.numel() == 0 || Q.stride(2) == 1, "the last dimension of Q must be contiguous");
    const int64_t rows = Q.size(0), heads = Q.size(1);
    // a dimension of one has any stride, and none that matters
    const int64_t row_stride = rows == 1 ? 0 : Q.stride(0), head_stride = heads == 1 ? 0 : Q.stride(1);
    c10::cuda::CUDAGuard guard(device);
    torch::Tensor O;
    if (out.has_value()) {
        O = *out;
        TORCH_CHECK(O.is_cuda() && O.device() == device && O.is_contiguous() && O.sizes() == Q.sizes() &&
                        O.scalar_type() == out_dtype,
                    "out must be a contiguous tensor of Q's shape and out_dtype on the pool's device");
    } else {
        O = new_tensor(Q.sizes(), out_dtype, device);
    }
    torch::Tensor L;
    if (want_lse) L = new_tensor({heads, rows}, torch::kFloat32, device);
    const int64_t capacity = block_table.size(1) * s.page_size;
    size_t bytes = 0;
    raise_status(lca_swa_cached_workspace_size(rows, heads, s.kv_heads, s.head_dim, batch, capacity, window_size,
                                               (int64_t)global_tokens.size(), &bytes),
                 "sliding_window_attention_cached");
    torch::Tensor ws;
    if (bytes > 0) ws = new_tensor({(int64_t)bytes}, torch::kUInt8, device);
    raise_status(lca_swa_forward_cached(Q.data_ptr(), type_code(Q.scalar_type(), "Q"), row_stride, head_stride, rows,
                                        heads, pool.data_ptr(), s.pages, s.kv_heads, s.page_size, s.head_dim,
                                        block_table.data_ptr<int32_t>(), batch, block_table.size(1),
                                        kv_lens.data_ptr<int32_t>(), cu_seqlens.data_ptr<int32_t>(), window_size,
                                        global_tokens.data(), (int64_t)global_tokens.size(), static_cast<float>(scale),
                                        O.data_ptr(), type_code(out_dtype, "out_dtype"),
                                        want_lse ? L.data_ptr<float>() : nullptr, bytes > 0 ? ws.data_ptr() : nullptr,
                                        bytes, current_stream()),
                 "sliding_window_attention_cached");
    if (want_lse) return {O, L};
    return {O};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.def("sliding_window_attention_forward", &sliding_window_attention_forward,
          "Sliding window + global token attention forward (B200 sm_100a)", py::arg("Q"), py::arg("K"),
          py::arg("V"), py::arg("window_size"), py::arg("global_tokens"), py::arg("scale"));
    m.def("sliding_window_attention_forward_list", &sliding_window_attention_forward_list,
          "As sliding_window_attention_forward, with global tokens as a list of ints", py::arg("Q"), py::arg("K"),
          py::arg("V"), py::arg("window_size"), py::arg("global_tokens"), py::arg("scale"));
    m.def("sliding_window_attention_forward_lse", &sliding_window_attention_forward_lse,
          "Forward returning (O, LSE); LSE is the natural-log log-sum-exp per query row", py::arg("Q"),
          py::arg("K"), py::arg("V"), py::arg("window_size"), py::arg("global_tokens"), py::arg("scale"));
    m.def("sliding_window_attention_forward_ex", &sliding_window_attention_forward_ex,
          "Forward with the output in out_dtype (float32, float16 or bfloat16), optionally causal (keys j <= i); "
          "returns [O] or [O, LSE]",
          py::arg("Q"), py::arg("K"), py::arg("V"), py::arg("window_size"), py::arg("global_tokens"),
          py::arg("scale"), py::arg("out_dtype"), py::arg("causal"), py::arg("want_lse"),
          py::arg("head_windows") = std::vector<int64_t>{}, py::arg("dilation") = 1,
          py::arg("cu_seqlens") = std::vector<int64_t>{}, py::arg("token_major") = false);
    m.def("sliding_window_attention_backward", &sliding_window_attention_backward,
          "Gradients (dQ, dK, dV), fp32, of the forward from its O and LSE and the gradient dO of O",
          py::arg("Q"), py::arg("K"), py::arg("V"), py::arg("O"), py::arg("LSE"), py::arg("dO"),
          py::arg("window_size"), py::arg("global_tokens"), py::arg("scale"));
    m.def("kv_cache_layout", &kv_cache_layout, "Block tables and slot maps of a step from its requests' lengths",
          py::arg("block_table"), py::arg("seq_lens"), py::arg("new_lens"), py::arg("free_pages"), py::arg("free_count"),
          py::arg("page_size"), py::arg("num_tokens"));
    m.def("kv_cache_release", &kv_cache_release, "Return the pages of the marked requests to the free list",
          py::arg("block_table"), py::arg("seq_lens"), py::arg("release"), py::arg("free_pages"), py::arg("free_count"),
          py::arg("page_size"));
    m.def("kv_cache_append", &kv_cache_append, "Quantise K and V rows into slots of a 4-bit pool", py::arg("pool"),
          py::arg("k"), py::arg("v"), py::arg("slots"));
    m.def("kv_cache_read", &kv_cache_read, "The values held in slots of a 4-bit pool", py::arg("pool"),
          py::arg("slots"), py::arg("out_dtype"));
    m.def("sliding_window_attention_cached", &sliding_window_attention_cached,
          "Causal sliding-window + global-token attention of new tokens over a 4-bit pool; returns [O] or [O, LSE]",
          py::arg("Q"), py::arg("pool"), py::arg("block_table"), py::arg("kv_lens"), py::arg("cu_seqlens"),
          py::arg("window_size"), py::arg("global_tokens"), py::arg("scale"), py::arg("out_dtype"), py::arg("want_lse"),
          py::arg("out") = py::none());
    m.def("device_error", &device_error, "Read and clear the device-side error word (synchronises)");
    m.attr("abi_version") = lca_abi_version();
}
