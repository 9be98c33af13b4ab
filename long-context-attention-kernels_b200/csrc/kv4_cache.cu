// kv4_cache.cu -- block tables and slot maps from request lengths, and the rows of the paged
// 4-bit KV cache: quantise-and-append, and read back.  The cache format is in kv4.h.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "kv4_attention.cuh"

namespace lca {
namespace kv4 {
namespace {

// ------------------------------------------------------------------ layout

// One block-wide exclusive scan of a value per thread, saturating at `cap` (cap < 2^31, so
// a sum of two saturated values fits 32 unsigned bits; min(a + b, cap) is associative for
// non-negative values).  `warp_sums` holds one word per warp.
template <int THREADS>
__device__ uint32_t scan_exclusive(uint32_t v, uint32_t cap, uint32_t* warp_sums, uint32_t* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t inc = min(v, cap);
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const uint32_t u = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc = min(inc + u, cap);
    }
    if (lane == 31) warp_sums[warp] = inc;
    __syncthreads();
    uint32_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
        if (w == warp) before = all;
        all = min(all + warp_sums[w], cap);
    }
    __syncthreads();
    *total = all;
    const uint32_t ex = __shfl_up_sync(0xffffffffu, inc, 1);
    return lane == 0 ? before : min(before + ex, cap);
}

constexpr int kLayoutThreads = 512;
constexpr int kLayoutRows = 4;  // consecutive rows per thread: 16-byte stores of slots and positions

__device__ __forceinline__ int32_t ceil_div(int32_t a, int32_t b) { return a / b + (a % b != 0); }

// Places new_lens[b] tokens behind seq_lens[b] for every request.  A request is placed whole or
// not at all: it needs its rows inside [0, rows), its pages inside its table row, and its
// new pages among the free ones, handed out from the end of the list in request order
// (a request that does not fit keeps its share of the order, so the outcome depends on the
// lengths alone).
//
// Bound by latency: every CTA scans the lengths of all requests for itself (two scans of at most
// kMaxRequests values, no traffic between CTAs and no second launch), then writes 16 bytes of
// slots and of positions per thread.  New table entries are written by the row that opens the
// page; entries that the scan reads and entries that it writes are never the same.
__global__ void __launch_bounds__(kLayoutThreads) kv_layout(const LayoutParams p) {
    extern __shared__ int32_t sm[];
    __shared__ uint32_t warp_sums[kLayoutThreads / 32];
    int32_t* s_end = sm;              // end of request b's rows
    int32_t* s_take = sm + p.batch;   // free pages handed out before b; -1: not placed
    ptx::griddep_wait();
    ptx::griddep_launch();
    const int per = (p.batch + kLayoutThreads - 1) / kLayoutThreads;
    const int b0 = threadIdx.x * per, b1 = min(b0 + per, p.batch);
    const int count = min(max(p.free_count[0], 0), p.free_cap);
    const uint32_t row_cap = (uint32_t)p.rows + 1, page_cap = (uint32_t)count + 1;

    uint32_t sum = 0;
    for (int b = b0; b < b1; ++b) sum = min(sum + min((uint32_t)max(p.new_lens[b], 0), row_cap), row_cap);
    uint32_t total;
    uint32_t end = scan_exclusive<kLayoutThreads>(sum, row_cap, warp_sums, &total);
    uint32_t pages = 0;
    for (int b = b0; b < b1; ++b) {
        const int have = max(p.seq_lens[b], 0), want = max(p.new_lens[b], 0);
        end = min(end + min((uint32_t)want, row_cap), row_cap);
        const bool fits = end <= (uint32_t)p.rows && (long long)have + want <= (long long)p.width * p.page_size;
        const int need = fits ? ceil_div(have + want, p.page_size) - ceil_div(have, p.page_size) : -1;
        s_end[b] = (int32_t)min(end, (uint32_t)p.rows);
        s_take[b] = need;
        pages = min(pages + (uint32_t)max(need, 0), page_cap);
    }
    uint32_t take = scan_exclusive<kLayoutThreads>(pages, page_cap, warp_sums, &total);
    uint32_t used = 0;
    for (int b = b0; b < b1; ++b) {
        const int need = s_take[b];
        const uint32_t before = take;
        take = min(take + (uint32_t)max(need, 0), page_cap);
        const bool ok = need == 0 || (need > 0 && take <= (uint32_t)count);
        s_take[b] = ok ? (int32_t)before : -1;
        used += ok ? (uint32_t)need : 0;
        if (blockIdx.x == 0) {
            const int have = max(p.seq_lens[b], 0), want = max(p.new_lens[b], 0);
            p.kv_lens[b] = ok ? have + want : 0;
            p.placed[b] = ok ? want : 0;
            p.next_seq_lens[b] = ok ? have + want : have;
            p.cu[b + 1] = s_end[b];
            if (b == 0) p.cu[0] = 0;
        }
    }
    if (blockIdx.x == 0) {
        scan_exclusive<kLayoutThreads>(used, page_cap, warp_sums, &total);
        if (threadIdx.x == 0) {
            p.next_free_count[0] = count - (int32_t)total;
            if (p.batch == 0) p.cu[0] = 0;
        }
    } else {
        __syncthreads();
    }

    for (long long r0 = ((long long)blockIdx.x * kLayoutThreads + threadIdx.x) * kLayoutRows; r0 < p.rows;
         r0 += (long long)gridDim.x * kLayoutThreads * kLayoutRows) {
        int lo = 0, hi = p.batch;  // the first request whose rows end behind r0
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (s_end[mid] > r0) hi = mid; else lo = mid + 1;
        }
        int slot[kLayoutRows], pos[kLayoutRows];
#pragma unroll
        for (int i = 0; i < kLayoutRows; ++i) {
            const int r = (int)r0 + i;
            slot[i] = pos[i] = -1;
            while (lo < p.batch && s_end[lo] <= r) ++lo;
            if (lo >= p.batch || s_take[lo] < 0) continue;
            const int have = max(p.seq_lens[lo], 0);
            const int at = have + r - (lo == 0 ? 0 : s_end[lo - 1]);
            const int pi = at / p.page_size, held = ceil_div(have, p.page_size), in = at - pi * p.page_size;
            int32_t* entry = p.table + (long long)lo * p.width + pi;
            int page;
            if (pi < held) {
                page = *entry;
            } else {
                page = p.free_pages[count - 1 - (s_take[lo] + pi - held)];
                if (in == 0) *entry = page;
            }
            const long long s = (long long)page * p.page_size + in;
            pos[i] = at;
            slot[i] = page >= 0 && s <= 0x7fffffffll ? (int)s : -1;
        }
        if (r0 + kLayoutRows <= p.rows) {
            *reinterpret_cast<int4*>(p.slots + r0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
            *reinterpret_cast<int4*>(p.positions + r0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
        } else {
            for (int i = 0; r0 + i < p.rows; ++i) {
                p.slots[r0 + i] = slot[i];
                p.positions[r0 + i] = pos[i];
            }
        }
    }
}

// Puts every page of the marked requests at the end of the free list, in request order, and
// sets their lengths to zero.  Same scan as kv_layout; the warps of the grid copy the rows.
__global__ void __launch_bounds__(kLayoutThreads) kv_release(const ReleaseParams p) {
    extern __shared__ int32_t sm[];
    __shared__ uint32_t warp_sums[kLayoutThreads / 32];
    ptx::griddep_wait();
    ptx::griddep_launch();
    const int per = (p.batch + kLayoutThreads - 1) / kLayoutThreads;
    const int b0 = threadIdx.x * per, b1 = min(b0 + per, p.batch);
    const int count = min(max(p.free_count[0], 0), p.free_cap);
    const uint32_t cap = (uint32_t)(p.free_cap - count);  // a list that is full drops the rest
    auto held = [&](int b) {
        if (!p.mask[b]) return 0;
        return min(ceil_div(max(p.seq_lens[b], 0), p.page_size), p.width);
    };
    uint32_t sum = 0, total;
    for (int b = b0; b < b1; ++b) sum = min(sum + (uint32_t)held(b), cap);
    uint32_t at = scan_exclusive<kLayoutThreads>(sum, cap, warp_sums, &total);
    for (int b = b0; b < b1; ++b) {
        sm[b] = (int32_t)at;
        at = min(at + (uint32_t)held(b), cap);
        if (blockIdx.x == 0) p.next_seq_lens[b] = p.mask[b] ? 0 : max(p.seq_lens[b], 0);
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) p.next_free_count[0] = count + (int32_t)total;
    __syncthreads();
    const int warps = kLayoutThreads / 32, lane = threadIdx.x & 31;
    for (int b = blockIdx.x * warps + (threadIdx.x >> 5); b < p.batch; b += gridDim.x * warps) {
        const int n = held(b), to = sm[b];
        for (int i = lane; i < n && to + i < (int)cap; i += 32)
            p.free_pages[count + to + i] = p.table[(long long)b * p.width + i];
    }
}

// ------------------------------------------------------------------ rows

template <typename T>
struct Half;  // the two 16-bit inputs: a pair of elements is a 32-bit word
template <>
struct Half<__half> {
    static constexpr uint32_t kSign = 0x80008000u;
    static __device__ __forceinline__ float low(uint32_t w) { return __half2float(__ushort_as_half((uint16_t)w)); }
    static __device__ __forceinline__ float high(uint32_t w) { return __half2float(__ushort_as_half((uint16_t)(w >> 16))); }
    static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {  // NaN if either is
        uint32_t d;
        asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
        return d;
    }
};
template <>
struct Half<__nv_bfloat16> {
    static constexpr uint32_t kSign = 0x80008000u;
    static __device__ __forceinline__ float low(uint32_t w) { return __uint_as_float(w << 16); }
    static __device__ __forceinline__ float high(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
    static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
        uint32_t d;
        asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
        return d;
    }
};

// Quantises one row held by LANES lanes, kPieces pieces of 8 elements (four pairs) a lane: the lane's
// words of codes, and the row's word of scale and zero point.  With lo = min(row, 0) and hi = max(row, 0): scale =
// hi/15 - lo/15 (products with fp32 1/15, so that opposite extremes of bf16 do not overflow) with
// its low four bits cleared, z = rint(-lo / scale), code = clamp(rint(x / scale) + z, 0, 15);
// quotients are fp32 products with 1 / scale.  Every operation is the IEEE one (no contraction), so
// the codes are a function of the row alone.  A scale below the smallest normal number stores
// zeros; a row with an infinity or a NaN stores NaN.
//
// The extremes are found on the 16-bit pairs, (max x, max -x) in one word across the lanes, so a
// step takes one shuffle and one instruction.  rint(y) for |y| < 2^22 is the sum with 1.5 * 2^23, whose
// low bits are the integer (rint and the conversion to int run at a quarter of that rate).
constexpr int kPieces = 2;

template <int LANES, typename T>
__device__ __forceinline__ void quantise(const uint32_t (&x)[4 * kPieces], uint32_t (&codes)[kPieces], uint32_t* word) {
    using H = Half<T>;
    uint32_t up = x[0], down = x[0] ^ H::kSign;
#pragma unroll
    for (int i = 1; i < 4 * kPieces; ++i) {
        up = H::max2(up, x[i]);
        down = H::max2(down, x[i] ^ H::kSign);
    }
    uint32_t ends = H::max2(__byte_perm(up, down, 0x5410), __byte_perm(up, down, 0x7632));
    ends = H::max2(ends, 0u);
#pragma unroll
    for (int o = LANES / 2; o > 0; o /= 2) ends = H::max2(ends, __shfl_xor_sync(0xffffffffu, ends, o));
    const float hi = H::low(ends), minus_lo = H::high(ends);
    constexpr float k15 = 1.0f / 15.0f, kMagic = 12582912.f;
    float scale = __fadd_rn(__fmul_rn(hi, k15), __fmul_rn(minus_lo, k15));
    scale = __uint_as_float(__float_as_uint(scale) & ~15u);
    const bool finite = hi < INFINITY && minus_lo < INFINITY;
    const bool normal = finite && scale >= 1.17549435e-38f;
    const float inv = normal ? __frcp_rn(scale) : 0.f;
    const float zm = normal ? __fadd_rn(__fmul_rn(minus_lo, inv), kMagic) : kMagic;  // kMagic + z
    const float z = __fsub_rn(zm, kMagic);
    const uint64_t magic2 = ptx::f2_pack(kMagic, kMagic), z2 = ptx::f2_pack(z, z);
#pragma unroll
    for (int piece = 0; piece < kPieces; ++piece) {
        uint32_t w = 0;
#pragma unroll
        for (int i = 4 * piece + 3; i >= 4 * piece; --i) {
            // the products one by one: a packed product and sum would be contracted into one operation
            const uint64_t y = ptx::f2_pack(__fmul_rn(H::low(x[i]), inv), __fmul_rn(H::high(x[i]), inv));
            const uint64_t c = ptx::f2_add(ptx::f2_add(y, magic2), z2);
            // never below 0: the least element rounds to -z itself
            w = w * 16u + __float_as_uint(fminf(ptx::f2_hi(c), kMagic + 15.f));
            w = w * 16u + __float_as_uint(fminf(ptx::f2_lo(c), kMagic + 15.f));
        }
        codes[piece] = normal ? w - 0x11111111u * 0x4b400000u : 0u;  // less the bits of kMagic in each
    }
    *word = normal ? __float_as_uint(scale) | (__float_as_uint(zm) & 15u) : (finite ? 0u : 0x7fc00000u);
}

constexpr int kRowThreads = 256;
struct Item {
    int token, head, row;
    uint8_t* block;  // NULL: a slot outside the pool
};

// Pair number `item` of the call.
template <int D>
__device__ __forceinline__ Item item_of(const RowsParams& p, long long item, long long items) {
    Item r = {0, 0, 0, nullptr};
    if (item >= items) return r;
    r.token = items <= 0x7fffffffll ? p.pool.per_token((int)item) : (int)(item / p.pool.kv_heads);
    r.head = (int)(item - (long long)r.token * p.pool.kv_heads);
    const int slot = p.slots[r.token];
    if (slot < 0) return r;
    const int block = slot / kBlock, page = p.pool.per_page(block);
    r.row = slot % kBlock;
    if (page < p.pool.pages)
        r.block = p.pool.data + (long long)((page * p.pool.kv_heads + r.head) * p.pool.page_blocks +
                                            block - page * p.pool.page_blocks) * block_bytes(D);
    return r;
}

// One group of d / 16 lanes per (token, head): a lane loads two pieces of 16 bytes of the K and of the V
// row and stores two 32-bit words of codes of each.  Bound by memory, 4d bytes read and d + 8 written
// a pair, as long as a row's reductions and its reciprocal are shared by 16 elements of a
// lane; with 8 the instructions bound it.  128K tokens of 8 heads of 128: 110 us, 94% of the copy rate;
// 155 us where rows are not on 16-byte boundaries (2-byte loads).
template <int D, typename T, bool VECTOR>
__global__ void __launch_bounds__(kRowThreads) kv4_append(const RowsParams p) {
    constexpr int LANES = D / (8 * kPieces), GROUPS = kRowThreads / LANES;
    const int lane = threadIdx.x % LANES;
    const long long items = (long long)p.rows * p.pool.kv_heads;
    const long long item = (long long)blockIdx.x * GROUPS + threadIdx.x / LANES;
    ptx::griddep_wait();
    ptx::griddep_launch();
    const Item at = item_of<D>(p, item, items);
    uint32_t x[2][4 * kPieces];
#pragma unroll
    for (int side = 0; side < 2; ++side) {
        const T* src = side == 0 ? static_cast<const T*>(p.k) + at.token * p.k_token + at.head * p.k_head
                                 : static_cast<const T*>(p.v) + at.token * p.v_token + at.head * p.v_head;
#pragma unroll
        for (int j = 0; j < kPieces; ++j) {
            uint4 a = make_uint4(0, 0, 0, 0);
            if (at.block != nullptr) {
                const T* from = src + 8 * (lane + LANES * j);
                if (VECTOR) {
                    a = *reinterpret_cast<const uint4*>(from);
                } else {
                    const uint16_t* e = reinterpret_cast<const uint16_t*>(from);
                    a = make_uint4(e[0] | (uint32_t)e[1] << 16, e[2] | (uint32_t)e[3] << 16, e[4] | (uint32_t)e[5] << 16,
                                   e[6] | (uint32_t)e[7] << 16);
                }
            }
            x[side][4 * j] = a.x, x[side][4 * j + 1] = a.y, x[side][4 * j + 2] = a.z, x[side][4 * j + 3] = a.w;
        }
    }
#pragma unroll
    for (int side = 0; side < 2; ++side) {
        uint32_t codes[kPieces], word;  // every lane takes part in the shuffles
        quantise<LANES, T>(x[side], codes, &word);
        if (at.block == nullptr) continue;
        uint32_t* to = reinterpret_cast<uint32_t*>(at.block + (side ? v_codes_at(D) : 0) + at.row * row_bytes(D)) + lane;
#pragma unroll
        for (int j = 0; j < kPieces; ++j) to[LANES * j] = codes[j];
        if (lane == side) *reinterpret_cast<uint32_t*>(at.block + (side ? v_words_at(D) : k_words_at(D)) + 4 * at.row) = word;
    }
}

template <typename T>
__device__ __forceinline__ void store8(T* to, const float (&x)[8]);
template <>
__device__ __forceinline__ void store8<float>(float* to, const float (&x)[8]) {
    reinterpret_cast<float4*>(to)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(to)[1] = make_float4(x[4], x[5], x[6], x[7]);
}
template <>
__device__ __forceinline__ void store8<__half>(__half* to, const float (&x)[8]) {
    __half2 h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
    *reinterpret_cast<uint4*>(to) = *reinterpret_cast<uint4*>(h);
}
template <>
__device__ __forceinline__ void store8<__nv_bfloat16>(__nv_bfloat16* to, const float (&x)[8]) {
    __nv_bfloat162 h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    *reinterpret_cast<uint4*>(to) = *reinterpret_cast<uint4*>(h);
}

// The eight values of a word of codes: c - z exactly in fp16 pairs, then one fp32 product each.
__device__ __forceinline__ void values_of(uint32_t codes, uint32_t word, float (&x)[8]) {
    const float scale = __uint_as_float(word & ~15u);
    const Zero z = zero_pair((word & 15u) * 0x10001u);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t pair = codes_pair(codes, i, z);  // elements i and i + 4
        const float2 c = __half22float2(*reinterpret_cast<const __half2*>(&pair));
        x[i] = __fmul_rn(scale, c.x);
        x[i + 4] = __fmul_rn(scale, c.y);
    }
}

// The rows of `slots` as values, rounded once to the output's type; a slot outside the pool reads
// as zeros.  The inverse of kv4_append, with the same lanes; bound by the bytes it writes.
constexpr int kReadItems = 2;  // pairs of a group of lanes, whose loads are in flight together

template <int D, typename T>
__global__ void __launch_bounds__(kRowThreads) kv4_read(const RowsParams p) {
    constexpr int LANES = D / (8 * kPieces), GROUPS = kRowThreads / LANES;
    const int lane = threadIdx.x % LANES;
    const long long items = (long long)p.rows * p.pool.kv_heads;
    const long long first = (long long)blockIdx.x * (GROUPS * kReadItems) + threadIdx.x / LANES;
    ptx::griddep_wait();
    ptx::griddep_launch();
    Item at[kReadItems];
    uint32_t codes[kReadItems][2][kPieces] = {}, words[kReadItems][2] = {};
#pragma unroll
    for (int i = 0; i < kReadItems; ++i) at[i] = item_of<D>(p, first + i * GROUPS, items);
#pragma unroll
    for (int i = 0; i < kReadItems; ++i) {
        if (at[i].block == nullptr) continue;
#pragma unroll
        for (int side = 0; side < 2; ++side) {
            const uint8_t* block = at[i].block;
            const uint32_t* from =
                reinterpret_cast<const uint32_t*>(block + (side ? v_codes_at(D) : 0) + at[i].row * row_bytes(D)) + lane;
#pragma unroll
            for (int j = 0; j < kPieces; ++j) codes[i][side][j] = from[LANES * j];
            words[i][side] = *reinterpret_cast<const uint32_t*>(block + (side ? v_words_at(D) : k_words_at(D)) + 4 * at[i].row);
        }
    }
#pragma unroll
    for (int i = 0; i < kReadItems; ++i) {
        if (first + i * GROUPS >= items) continue;
#pragma unroll
        for (int side = 0; side < 2; ++side) {
            T* to = side == 0 ? static_cast<T*>(p.k) + at[i].token * p.k_token + at[i].head * p.k_head
                              : static_cast<T*>(p.v) + at[i].token * p.v_token + at[i].head * p.v_head;
#pragma unroll
            for (int j = 0; j < kPieces; ++j) {
                float x[8];
                values_of(codes[i][side][j], words[i][side], x);
                store8<T>(to + 8 * (lane + LANES * j), x);
            }
        }
    }
}

unsigned row_blocks(int d, int each, const RowsParams& p) {
    const long long pairs = kRowThreads / (d / (8 * kPieces)) * each;
    return (unsigned)(((long long)p.rows * p.pool.kv_heads + pairs - 1) / pairs);
}

template <int D, typename T>
cudaError_t append_of(bool vector, const RowsParams& p, cudaStream_t stream) {
    return launch_early(vector ? kv4_append<D, T, true> : kv4_append<D, T, false>, dim3(row_blocks(D, 1, p)), kRowThreads, 0,
                        stream, p);
}

template <int D>
cudaError_t read_of(int out_dtype, const RowsParams& p, cudaStream_t stream) {
    auto kernel = out_dtype == LCA_DTYPE_F32 ? kv4_read<D, float>
                                             : (out_dtype == LCA_DTYPE_F16 ? kv4_read<D, __half> : kv4_read<D, __nv_bfloat16>);
    return launch_early(kernel, dim3(row_blocks(D, kReadItems, p)), kRowThreads, 0, stream, p);
}

}  // namespace

cudaError_t launch_layout(const LayoutParams& p, cudaStream_t stream) {
    const int blocks = std::max(1, std::min(148, (p.rows + kLayoutThreads * kLayoutRows - 1) /
                                                     (kLayoutThreads * kLayoutRows)));
    const size_t smem = 2 * sizeof(int32_t) * (size_t)p.batch;
    static_assert(2 * sizeof(int32_t) * kMaxRequests <= 64 * 1024, "shared memory of the scan");
    if (smem > 40 * 1024) {
        cudaError_t e = cudaFuncSetAttribute(kv_layout, cudaFuncAttributeMaxDynamicSharedMemorySize, 64 * 1024);
        if (e != cudaSuccess) return e;
    }
    return launch_early(kv_layout, dim3(blocks), kLayoutThreads, smem, stream, p);
}

cudaError_t launch_release(const ReleaseParams& p, cudaStream_t stream) {
    const int blocks = std::max(1, std::min(148, (p.batch + kLayoutThreads / 32 - 1) / (kLayoutThreads / 32)));
    static_assert(sizeof(int32_t) * kMaxRequests <= 40 * 1024, "shared memory of the scan");
    return launch_early(kv_release, dim3(blocks), kLayoutThreads, sizeof(int32_t) * (size_t)p.batch, stream, p);
}

cudaError_t launch_append(int d, int dtype, bool vector, const RowsParams& p, cudaStream_t stream) {
    if (d == 64)
        return dtype == LCA_DTYPE_F16 ? append_of<64, __half>(vector, p, stream)
                                      : append_of<64, __nv_bfloat16>(vector, p, stream);
    return dtype == LCA_DTYPE_F16 ? append_of<128, __half>(vector, p, stream)
                                  : append_of<128, __nv_bfloat16>(vector, p, stream);
}

cudaError_t launch_read(int d, int out_dtype, const RowsParams& p, cudaStream_t stream) {
    return d == 64 ? read_of<64>(out_dtype, p, stream) : read_of<128>(out_dtype, p, stream);
}

}  // namespace kv4
}  // namespace lca
