// kv4_capi.cpp -- the C ABI of the paged 4-bit KV cache (include/lca.h): argument checks and
// launches.  Nothing here allocates device memory or synchronises.
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>

#include "kv4.h"
#include "lca.h"
#include "swa_kernels.h"

namespace {

using lca::report_error;

constexpr int64_t kMaxRows = (int64_t)1 << 30;

bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

int after_launch(cudaError_t e, const char* what) {
    if (e == cudaSuccess) return LCA_OK;
    return report_error(LCA_ERR_CUDA, "%s: %s (%s)", what, cudaGetErrorName(e), cudaGetErrorString(e));
}

int check_device(int** err_word = nullptr, unsigned long long* wait_ns = nullptr) {
    int* err = nullptr;
    unsigned long long ns = 0;
    const int st = lca::device_info(&err, &ns);
    if (err_word != nullptr) *err_word = err;
    if (wait_ns != nullptr) *wait_ns = ns;
    return st;
}

size_t round256(size_t n) { return (n + 255) / 256 * 256; }

int check_heads(int64_t rows, int64_t heads, int64_t kv_heads) {
    if (kv_heads < 1 || heads < 1 || heads % kv_heads != 0 || heads > 65535)
        return report_error(LCA_ERR_INVALID_ARGUMENT, "heads (%lld) must be a multiple of kv_heads (%lld), at most 65535",
                            (long long)heads, (long long)kv_heads);
    if (rows > INT_MAX / heads)
        return report_error(LCA_ERR_UNSUPPORTED, "%lld rows of %lld heads are too many", (long long)rows, (long long)heads);
    return LCA_OK;
}

int check_page_size(int64_t page_size) {
    if (page_size <= 0 || page_size % lca::kv4::kBlock != 0 || page_size > 65536)
        return report_error(LCA_ERR_INVALID_ARGUMENT, "page_size must be a multiple of %d up to 65536 (got %lld)",
                            lca::kv4::kBlock, (long long)page_size);
    return LCA_OK;
}

int check_table(int64_t batch, int64_t width, int64_t page_size) {
    if (batch < 0 || width < 0) return report_error(LCA_ERR_INVALID_ARGUMENT, "negative shape of block_table");
    if (batch > lca::kv4::kMaxRequests)
        return report_error(LCA_ERR_UNSUPPORTED, "%lld requests are more than %d", (long long)batch,
                            lca::kv4::kMaxRequests);
    if (width > ((int64_t)1 << 30) / page_size)
        return report_error(LCA_ERR_UNSUPPORTED, "block_table holds %lld pages of %lld tokens a request (at most 2^30 tokens)",
                            (long long)width, (long long)page_size);
    return LCA_OK;
}

int check_pool(lca::kv4::Pool* pool, const void* data, int64_t pages, int64_t kv_heads, int64_t page_size,
               int64_t head_dim) {
    if (head_dim != 64 && head_dim != 128)
        return report_error(LCA_ERR_UNSUPPORTED, "head_dim %lld is not supported (64 or 128)", (long long)head_dim);
    if (int st = check_page_size(page_size)) return st;
    if (pages < 0 || kv_heads < 1 || kv_heads > 65535)
        return report_error(LCA_ERR_INVALID_ARGUMENT, "the pool needs pages >= 0 and 1 to 65535 kv_heads (got %lld and %lld)",
                            (long long)pages, (long long)kv_heads);
    if (pages > INT_MAX / page_size)
        return report_error(LCA_ERR_UNSUPPORTED, "the pool holds more than 2^31 - 1 tokens");
    if (pages > 0 && data == nullptr) return report_error(LCA_ERR_INVALID_ARGUMENT, "pool must be non-NULL");
    if (!aligned(data, 16)) return report_error(LCA_ERR_INVALID_ARGUMENT, "pool must be 16-byte aligned");
    pool->data = static_cast<uint8_t*>(const_cast<void*>(data));
    pool->pages = (int)pages;
    pool->kv_heads = (int)kv_heads;
    pool->page_blocks = (int)(page_size / lca::kv4::kBlock);
    pool->per_page = lca::kv4::Divisor((uint32_t)pool->page_blocks);
    pool->per_token = lca::kv4::Divisor((uint32_t)kv_heads);
    return LCA_OK;
}

int check_input_type(int dtype) {
    if (dtype != LCA_DTYPE_F16 && dtype != LCA_DTYPE_BF16)
        return report_error(LCA_ERR_UNSUPPORTED, "dtype %d is not supported (fp16 or bf16 inputs)", dtype);
    return LCA_OK;
}

int check_out_type(int dtype) {
    if (dtype != LCA_DTYPE_F16 && dtype != LCA_DTYPE_BF16 && dtype != LCA_DTYPE_F32)
        return report_error(LCA_ERR_UNSUPPORTED, "out_dtype %d is not supported (fp32, fp16 or bf16)", dtype);
    return LCA_OK;
}

int check_rows(int64_t rows, int64_t heads) {
    if (rows < 0) return report_error(LCA_ERR_INVALID_ARGUMENT, "negative row count %lld", (long long)rows);
    if (rows > kMaxRows || rows * heads > ((int64_t)1 << 34))
        return report_error(LCA_ERR_UNSUPPORTED, "%lld rows of %lld heads are too many", (long long)rows, (long long)heads);
    return LCA_OK;
}

}  // namespace

extern "C" {

int lca_kv_layout(int32_t* block_table, int64_t batch, int64_t table_width, const int32_t* seq_lens,
                  const int32_t* new_lens, const int32_t* free_pages, int64_t free_capacity,
                  const int32_t* free_count, int64_t page_size, int64_t num_tokens, int32_t* slots,
                  int32_t* positions, int32_t* cu_seqlens, int32_t* kv_lens, int32_t* placed,
                  int32_t* next_seq_lens, int32_t* next_free_count, void* stream) {
    if (int st = check_page_size(page_size)) return st;
    if (int st = check_table(batch, table_width, page_size)) return st;
    if (int st = check_rows(num_tokens, 1)) return st;
    if (free_capacity < 0 || free_capacity > kMaxRows)
        return report_error(LCA_ERR_INVALID_ARGUMENT, "free_capacity %lld is outside [0, 2^30]", (long long)free_capacity);
    const bool some = batch > 0;
    if (cu_seqlens == nullptr || free_count == nullptr || next_free_count == nullptr ||
        (num_tokens > 0 && (slots == nullptr || positions == nullptr)) || (free_capacity > 0 && free_pages == nullptr) ||
        (some && (seq_lens == nullptr || new_lens == nullptr || kv_lens == nullptr || placed == nullptr ||
                  next_seq_lens == nullptr)) ||
        (some && table_width > 0 && block_table == nullptr))
        return report_error(LCA_ERR_INVALID_ARGUMENT, "the layout's arrays must be non-NULL");
    if (!aligned(slots, 16) || !aligned(positions, 16))
        return report_error(LCA_ERR_INVALID_ARGUMENT, "slots and positions must be 16-byte aligned");
    if ((some && next_seq_lens == seq_lens) || next_free_count == free_count)
        return report_error(LCA_ERR_INVALID_ARGUMENT, "the next lengths and free count must not overwrite the present ones");
    if (int st = check_device()) return st;
    lca::kv4::LayoutParams p;
    p.table = block_table;
    p.batch = (int)batch;
    p.width = (int)table_width;
    p.page_size = (int)page_size;
    p.rows = (int)num_tokens;
    p.seq_lens = seq_lens;
    p.new_lens = new_lens;
    p.free_pages = free_pages;
    p.free_count = free_count;
    p.free_cap = (int)free_capacity;
    p.slots = slots;
    p.positions = positions;
    p.cu = cu_seqlens;
    p.kv_lens = kv_lens;
    p.placed = placed;
    p.next_seq_lens = next_seq_lens;
    p.next_free_count = next_free_count;
    return after_launch(lca::kv4::launch_layout(p, static_cast<cudaStream_t>(stream)), "layout launch");
}

int lca_kv_release(const int32_t* block_table, int64_t batch, int64_t table_width, const int32_t* seq_lens,
                   const uint8_t* release, int32_t* free_pages, int64_t free_capacity, const int32_t* free_count,
                   int64_t page_size, int32_t* next_seq_lens, int32_t* next_free_count, void* stream) {
    if (int st = check_page_size(page_size)) return st;
    if (int st = check_table(batch, table_width, page_size)) return st;
    if (free_capacity < 0 || free_capacity > kMaxRows)
        return report_error(LCA_ERR_INVALID_ARGUMENT, "free_capacity %lld is outside [0, 2^30]", (long long)free_capacity);
    const bool some = batch > 0;
    if (free_count == nullptr || next_free_count == nullptr || (free_capacity > 0 && free_pages == nullptr) ||
        (some && (seq_lens == nullptr || release == nullptr || next_seq_lens == nullptr)) ||
        (some && table_width > 0 && block_table == nullptr))
        return report_error(LCA_ERR_INVALID_ARGUMENT, "the release's arrays must be non-NULL");
    if ((some && next_seq_lens == seq_lens) || next_free_count == free_count)
        return report_error(LCA_ERR_INVALID_ARGUMENT, "the next lengths and free count must not overwrite the present ones");
    if (int st = check_device()) return st;
    lca::kv4::ReleaseParams p;
    p.table = block_table;
    p.batch = (int)batch;
    p.width = (int)table_width;
    p.page_size = (int)page_size;
    p.seq_lens = seq_lens;
    p.mask = release;
    p.free_pages = free_pages;
    p.free_cap = (int)free_capacity;
    p.free_count = free_count;
    p.next_seq_lens = next_seq_lens;
    p.next_free_count = next_free_count;
    return after_launch(lca::kv4::launch_release(p, static_cast<cudaStream_t>(stream)), "release launch");
}

int lca_kv4_append(void* pool, int64_t num_pages, int64_t kv_heads, int64_t page_size, int64_t head_dim, const void* k,
                   const void* v, int dtype, int64_t k_token_stride, int64_t k_head_stride, int64_t v_token_stride,
                   int64_t v_head_stride, const int32_t* slots, int64_t num_tokens, void* stream) {
    lca::kv4::RowsParams p;
    if (int st = check_input_type(dtype)) return st;
    if (int st = check_pool(&p.pool, pool, num_pages, kv_heads, page_size, head_dim)) return st;
    if (int st = check_rows(num_tokens, kv_heads)) return st;
    if (num_tokens == 0 || num_pages == 0) return LCA_OK;
    if (k == nullptr || v == nullptr || slots == nullptr)
        return report_error(LCA_ERR_INVALID_ARGUMENT, "k, v and slots must be non-NULL");
    if (!aligned(k, 2) || !aligned(v, 2)) return report_error(LCA_ERR_INVALID_ARGUMENT, "k and v must be 2-byte aligned");
    if (int st = check_device()) return st;
    const bool vector = aligned(k, 16) && aligned(v, 16) &&
                        ((k_token_stride | k_head_stride | v_token_stride | v_head_stride) & 7) == 0;
    p.k = const_cast<void*>(k);
    p.v = const_cast<void*>(v);
    p.k_token = k_token_stride;
    p.k_head = k_head_stride;
    p.v_token = v_token_stride;
    p.v_head = v_head_stride;
    p.slots = slots;
    p.rows = (int)num_tokens;
    return after_launch(lca::kv4::launch_append((int)head_dim, dtype, vector, p, static_cast<cudaStream_t>(stream)),
                        "append launch");
}

int lca_kv4_read(const void* pool, int64_t num_pages, int64_t kv_heads, int64_t page_size, int64_t head_dim,
                 const int32_t* slots, int64_t num_tokens, void* k, void* v, int out_dtype, void* stream) {
    lca::kv4::RowsParams p;
    if (int st = check_out_type(out_dtype)) return st;
    if (int st = check_pool(&p.pool, pool, num_pages, kv_heads, page_size, head_dim)) return st;
    if (int st = check_rows(num_tokens, kv_heads)) return st;
    if (num_tokens == 0) return LCA_OK;
    if (k == nullptr || v == nullptr || slots == nullptr)
        return report_error(LCA_ERR_INVALID_ARGUMENT, "k, v and slots must be non-NULL");
    if (!aligned(k, 16) || !aligned(v, 16))
        return report_error(LCA_ERR_INVALID_ARGUMENT, "k and v must be 16-byte aligned");
    if (int st = check_device()) return st;
    p.k = k;
    p.v = v;
    p.k_token = p.v_token = kv_heads * head_dim;
    p.k_head = p.v_head = head_dim;
    p.slots = slots;
    p.rows = (int)num_tokens;
    return after_launch(lca::kv4::launch_read((int)head_dim, out_dtype, p, static_cast<cudaStream_t>(stream)),
                        "read launch");
}

int lca_swa_cached_workspace_size(int64_t num_rows, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t batch,
                                  int64_t capacity, int64_t window_size, int64_t num_unique_global, size_t* out_bytes) {
    if (out_bytes == nullptr) return report_error(LCA_ERR_INVALID_ARGUMENT, "out_bytes is NULL");
    *out_bytes = 0;
    if (window_size < 0)
        return report_error(LCA_ERR_INVALID_ARGUMENT, "window_size must be >= 0 (got %lld)", (long long)window_size);
    if (num_rows < 0 || batch < 0 || capacity < 0 || num_unique_global < 0)
        return report_error(LCA_ERR_INVALID_ARGUMENT, "negative shape");
    if (int st = check_heads(num_rows, heads, kv_heads)) return st;
    const lca::kv4::AttnPlan a =
        lca::kv4::plan_attention(num_rows, heads, kv_heads, head_dim, batch, capacity, window_size, num_unique_global);
    *out_bytes = round256(a.part_o) + round256(a.part_ml) + a.cuts;
    return LCA_OK;
}

int lca_swa_forward_cached(const void* q, int dtype, int64_t q_row_stride, int64_t q_head_stride, int64_t num_rows,
                           int64_t heads, const void* pool, int64_t num_pages, int64_t kv_heads, int64_t page_size,
                           int64_t head_dim, const int32_t* block_table, int64_t batch, int64_t table_width,
                           const int32_t* kv_lens, const int32_t* cu_seqlens, int64_t window_size,
                           const int64_t* global_tokens, int64_t num_global_tokens, float scale, void* out,
                           int out_dtype, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
    lca::kv4::AttnParams p;
    if (int st = check_input_type(dtype)) return st;
    if (int st = check_out_type(out_dtype)) return st;
    if (int st = check_pool(&p.pool, pool, num_pages, kv_heads, page_size, head_dim)) return st;
    if (int st = check_table(batch, table_width, page_size)) return st;
    if (int st = check_rows(num_rows, heads)) return st;
    if (int st = check_heads(num_rows, heads, kv_heads)) return st;
    if (window_size < 0)
        return report_error(LCA_ERR_INVALID_ARGUMENT, "window_size must be >= 0 (got %lld)", (long long)window_size);
    if (num_global_tokens < 0 || (num_global_tokens > 0 && global_tokens == nullptr))
        return report_error(LCA_ERR_INVALID_ARGUMENT, "global_tokens is NULL or its count negative");
    const int64_t capacity = table_width * page_size;
    lca::kv4::Globals g;
    int n = 0;
    for (int64_t i = 0; i < num_global_tokens; ++i) {
        const int64_t t = global_tokens[i];
        if (t < 0 || t >= std::max<int64_t>(capacity, 1))
            return report_error(LCA_ERR_INDEX, "global token %lld is outside a request's capacity of %lld tokens",
                                (long long)t, (long long)capacity);
        int at = (int)(std::lower_bound(g.at, g.at + n, (int32_t)t) - g.at);
        if (at < n && g.at[at] == (int32_t)t) continue;
        if (n == lca::kv4::kMaxGlobals)
            return report_error(LCA_ERR_UNSUPPORTED, "more than %d distinct global tokens", lca::kv4::kMaxGlobals);
        std::copy_backward(g.at + at, g.at + n, g.at + n + 1);
        g.at[at] = (int32_t)t;
        ++n;
    }
    if (num_rows == 0 || batch == 0) return LCA_OK;
    if (q == nullptr || out == nullptr || kv_lens == nullptr || cu_seqlens == nullptr ||
        (table_width > 0 && block_table == nullptr))
        return report_error(LCA_ERR_INVALID_ARGUMENT, "q, out, block_table, kv_lens and cu_seqlens must be non-NULL");
    if (!aligned(q, 16) || ((q_row_stride | q_head_stride) & 7) != 0)
        return report_error(LCA_ERR_INVALID_ARGUMENT, "q must be 16-byte aligned with strides of a multiple of 8 elements");
    if (!aligned(out, 16)) return report_error(LCA_ERR_INVALID_ARGUMENT, "out must be 16-byte aligned");
    if (!aligned(lse, 4)) return report_error(LCA_ERR_INVALID_ARGUMENT, "lse must be 4-byte aligned");
    const lca::kv4::AttnPlan a =
        lca::kv4::plan_attention(num_rows, heads, kv_heads, head_dim, batch, capacity, window_size, n);
    const size_t need = round256(a.part_o) + round256(a.part_ml) + a.cuts;
    if (need > 0 && (workspace == nullptr || !aligned(workspace, 256) || workspace_bytes < need))
        return report_error(LCA_ERR_WORKSPACE, "workspace needs %zu bytes, non-NULL and 256-byte aligned (got %zu)", need,
                            workspace_bytes);
    if (int st = check_device(&p.err_word, &p.wait_ns)) return st;
    p.ctas = a.ctas;
    p.min_tiles = a.min_tiles;
    p.split = a.split;
    p.items = a.items;
    p.part_o = static_cast<float*>(workspace);
    uint8_t* at = static_cast<uint8_t*>(workspace) + round256(a.part_o);
    p.part_ml = reinterpret_cast<float2*>(at);
    p.cuts = a.cuts > 0 ? reinterpret_cast<lca::kv4::Cut*>(at + round256(a.part_ml)) : nullptr;
    p.bf16 = dtype == LCA_DTYPE_BF16;
    p.out_dtype = out_dtype;
    p.q = q;
    p.q_token = q_row_stride;
    p.q_head = q_head_stride;
    p.table = block_table;
    p.kv_lens = kv_lens;
    p.cu = cu_seqlens;
    p.batch = (int)batch;
    p.width = (int)table_width;
    p.rows = (int)num_rows;
    p.heads = (int)heads;
    p.group = (int)(heads / kv_heads);
    p.per_group = lca::kv4::Divisor((uint32_t)p.group);
    p.window = (int)std::min<int64_t>(window_size, (int64_t)1 << 30);
    p.num_globals = n;
    p.scale = scale;
    p.out = out;
    p.lse = lse;
    return after_launch(lca::kv4::launch_attention((int)head_dim, a.tile_rows, a.tile_keys, p, g,
                                                   static_cast<cudaStream_t>(stream)),
                        "cached attention launch");
}

}  // extern "C"
