// kv4.h -- internal interface between the C-ABI layer (kv4_capi.cpp) and the kernels of the
// paged 4-bit KV cache (kv4_cache.cu, kv4_attention.cu, kv4_chunk.cu).  Not part of the public ABI.
//
// Cache format.  A pool is [pages][kv_heads] pieces of page_size tokens; a piece is
// page_size / 16 blocks, and a block holds 16 tokens of one head contiguously:
//
//   K codes [16][d / 2] | V codes [16][d / 2] | K words [16] | V words [16]   = 16 * (d + 8) bytes
//
// so one block (or every block of a page) is one bulk copy.  Bits 4j .. 4j+3 of code word i
// of a row hold element 8i + j.  A row's word is its fp32 scale with the zero point z in the
// low four bits; an element is scale * (code - z).
#pragma once

#include <cuda_runtime.h>
#include <cstdint>

#include "lca.h"

namespace lca {
namespace kv4 {

constexpr int kBlock = 16;             // tokens per block
constexpr int kMaxGlobals = 1024;      // global tokens of one attention call (kernel parameter space)
constexpr int kChunkRows = 256;        // query rows and keys of a tile of the tcgen05 kernel
constexpr int kChunkKeys = 64;
constexpr int kMaxRequests = 8192;     // requests of one layout call (shared memory of its scan)

__host__ __device__ constexpr int row_bytes(int d) { return d / 2; }              // code bytes of one row
__host__ __device__ constexpr int block_bytes(int d) { return kBlock * (d + 8); }
__host__ __device__ constexpr int v_codes_at(int d) { return kBlock * d / 2; }
__host__ __device__ constexpr int k_words_at(int d) { return kBlock * d; }
__host__ __device__ constexpr int v_words_at(int d) { return kBlock * d + 4 * kBlock; }

// Division by a number that a call fixes, as a multiplication (Granlund and Montgomery 1994): for n and
// d below 2^31, n / d = (n + floor(n m / 2^32)) >> s with s = ceil(log2 d), m = floor(2^32 (2^s - d) / d)
// + 1.
struct Divisor {
    uint32_t d, m, s;
    explicit Divisor(uint32_t by = 1) : d(by), m(1), s(0) {
        while ((1ull << s) < by) ++s;
        m = (uint32_t)(((1ull << 32) * ((1ull << s) - by)) / by + 1);
    }
#ifdef __CUDACC__
    __device__ __forceinline__ int operator()(int n) const {
        return (int)((__umulhi((uint32_t)n, m) + (uint32_t)n) >> s);
    }
#endif
};

struct Pool {
    uint8_t* data;
    int pages, kv_heads;
    int page_blocks;  // page_size / 16
    Divisor per_page, per_token;  // by page_blocks, by kv_heads
};

struct LayoutParams {
    int32_t* table;  // [batch][width]
    int batch, width, page_size, rows;
    const int32_t *seq_lens, *new_lens, *free_pages, *free_count;
    int free_cap;
    int32_t *slots, *positions, *cu, *kv_lens, *placed, *next_seq_lens, *next_free_count;
};

struct ReleaseParams {
    const int32_t* table;
    int batch, width, page_size;
    const int32_t* seq_lens;
    const uint8_t* mask;
    int32_t* free_pages;
    int free_cap;
    const int32_t* free_count;
    int32_t *next_seq_lens, *next_free_count;
};

struct RowsParams {  // append (k, v read) and read (k, v written)
    Pool pool;
    void *k, *v;
    long long k_token, k_head, v_token, v_head;  // strides in elements
    const int32_t* slots;
    int rows;
};

struct Globals {
    int32_t at[kMaxGlobals];  // sorted, unique
};

// An item that its first CTA could not finish: what the merge has to know of it.
struct Cut {
    long long end, per;    // the end of the item on the line of tiles, and a CTA's share of that; end 0: no item
    int slot;              // of the first part, in the first CTA's two
    int q0, rows, head, q_tile;
};

struct AttnParams {
    Pool pool;
    const void* q;
    long long q_token, q_head;  // strides in elements
    const int32_t *table, *kv_lens, *cu;
    int batch, width;
    int rows, heads, group;  // query rows, query heads, query heads per KV head
    Divisor per_group;
    int window, num_globals;
    float scale;
    int bf16, out_dtype;
    void* out;   // [rows][heads][d]
    float* lse;  // [heads][rows] or NULL
    int ctas, split;  // CTAs that share the line of tiles; whether items may be cut between them
    int min_tiles;    // and then the least tiles of a CTA
    long long items;  // at most this many items
    float* part_o;    // [ctas][2][tile rows][d]: the parts of cut items, and
    float2* part_ml;  // [ctas][2][tile rows]: their maxima and sums
    Cut* cuts;        // [ctas], or NULL: the merge finds the items itself
    int* err_word;
    unsigned long long wait_ns;
};

struct AttnPlan {
    int tile_rows;  // query rows of an item: 8, 16 or 32 (kv4_attention.cu) or kChunkRows (kv4_chunk.cu)
    int tile_keys;  // keys of a tile
    int ctas, min_tiles;
    bool split;
    int64_t items;
    size_t part_o, part_ml, cuts;  // bytes
};

cudaError_t launch_layout(const LayoutParams& p, cudaStream_t stream);
cudaError_t launch_release(const ReleaseParams& p, cudaStream_t stream);
cudaError_t launch_append(int d, int dtype, bool vector, const RowsParams& p, cudaStream_t stream);
cudaError_t launch_read(int d, int out_dtype, const RowsParams& p, cudaStream_t stream);
AttnPlan plan_attention(int64_t rows, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t batch, int64_t capacity,
                        int64_t window, int64_t num_globals);
cudaError_t launch_chunk(int d, const AttnParams& p, const Globals& g, cudaStream_t stream);
cudaError_t launch_attention(int d, int tile_rows, int tile_keys, const AttnParams& p, const Globals& g,
                             cudaStream_t stream);

}  // namespace kv4

// capi.cpp: checks the current device; its error word and wait limit.
int device_info(int** err_word, unsigned long long* wait_ns);

}  // namespace lca
