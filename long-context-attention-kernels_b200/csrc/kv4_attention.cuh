// kv4_attention.cuh -- what the two kernels of attention over the paged 4-bit KV cache share: the
// unpacking of codes and the division of a call's work (kv4_attention.cu: few query rows a
// request, streamed; kv4_chunk.cu: many, on tcgen05).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>
#include <cstdlib>
#include <utility>

#include "kv4.h"
#include "sm100_ptx.cuh"

namespace lca {
namespace kv4 {

constexpr uint32_t kAll = 0xffffffffu;

// A value that every lane holds alike, in a form from which the compiler can tell (branches on
// it need no reconvergence, addresses go to uniform registers).
__device__ __forceinline__ int uniform(int v) { return __shfl_sync(kAll, v, 0); }

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// The range of the weights.  A weight enters the second product as fp16, as w_j = 2^(y_j - M) with y_j = x_j
// log2(e) + log2(sv_j), and where the output is finer than bf16 the remainder w_j - fp16(w_j) follows as
// another fp16.  fp16 has no step below 2^-24, so a long tail of small weights would vanish if the largest
// were 1: M is taken kHead below the running maximum of y, and moves once y has passed it by kRise, so the
// largest weight of a row is at least 2^kHead and none passes 2^kRise = 61147 of fp16's 65504.  Two halves are
// off by at most 2^-22 of w_j, or 2^-33 of the row's largest weight where that is more; one half by 2^-11 of w_j
// instead of the 2^-22.  A greater kHead leaves less room before M has to move: 9 gains a factor 2 and takes
// 157 us instead of 154 for four chunks of 2K (bf16, 32 / 8 heads of 128, window 512).
// The sum takes p_j = w_j / sv_j; log2(sv) is cut off at kLeast, so that 2^30 of them stay in fp32's range.
constexpr float kHead = 8.f, kRise = 15.9f, kLeast = -80.f;

// The square root of 2^d, d <= 0.  M is up to 200 apart between keys whose V is near zero and keys whose V is
// large; 2^d itself would be 0 then, while a sum of the former, 2^80 times larger, still counts.
__device__ __forceinline__ float ex2_half(float d) { return ptx::ex2(0.5f * d); }

// The natural logarithm of a row's sum l 2^m.
__device__ __forceinline__ float lse_of(float m, float l) {
    constexpr float kTakeOff = 1.f / 256.f;
    static_assert(kHead == 8.f, "kTakeOff is 2^-kHead");
    return l == 0.f ? -INFINITY : ((m + kHead) + log2f(l * kTakeOff)) * kLn2;
}

__device__ __forceinline__ int lower_bound(const int32_t* a, int n, int v) {
    // the usual answers first: the globals lie at the start of long contexts
    if (n == 0 || v <= a[0]) return 0;
    if (v > a[n - 1]) return n;
    int lo = 0;
    while (lo < n) {
        const int mid = (lo + n) >> 1;
        if (a[mid] < v) lo = mid + 1; else n = mid;
    }
    return lo;
}

__device__ __forceinline__ float lg2(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint32_t hsub2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}

__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}

__device__ __forceinline__ uint32_t hfma2(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t d;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
}

// Two codes minus their zero points as a pair of fp16, from the nibbles at bits 0 and 16 (LOW) or 4
// and 20 of w.  0x6400 | c is 1024 + c; 0x6400 | 16 c is 1024 + 16 c, a sixteenth of which is 64 + c.
// z holds the fp16 pairs 1024 + zp and -(64 + zp); every step is exact.
struct Zero {
    uint32_t low, high;
};

// z: a zero point in bits 0 .. 3 and one in bits 16 .. 19.
__device__ __forceinline__ Zero zero_pair(uint32_t z) { return {0x64006400u + z, 0xd400d400u + 16u * z}; }

__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t b, uint32_t c) {  // (a & b) | c, one instruction
    uint32_t d;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
}

__device__ __forceinline__ uint32_t codes_low(uint32_t w, const Zero& z) {
    return hsub2(and_or(w, 0x000f000fu, 0x64006400u), z.low);
}

__device__ __forceinline__ uint32_t codes_high(uint32_t w, const Zero& z) {
    return hfma2(and_or(w, 0x00f000f0u, 0x64006400u), 0x2c002c00u, z.high);
}

__device__ __forceinline__ uint32_t codes_pair(uint32_t w, int nibble, const Zero& z) {  // nibble: 0 .. 3, a constant
    const uint32_t v = nibble >= 2 ? w >> 8 : w;
    return (nibble & 1) ? codes_high(v, z) : codes_low(v, z);
}

// ------------------------------------------------------------------ the work of a call

// An item is one (request, KV head, tile of ROWS query rows); rows of a request are ordered
// token by token, and within a token by the query heads of the group.  Its keys are whole
// tiles of TILE positions that cover the band of its rows, then tiles of TILE gathered
// global tokens in front of the band.  Request b has `items` items of at most `tiles` tiles
// each (exactly `tiles` when it has one query tile per head); all its tiles, item after item and
// request after request, form one line of tiles that the CTAs share out evenly.
struct Request {
    int q0, len, rows;      // first row of q, cached tokens, rows (tokens * group)
    int q_tiles, tiles;
};

struct Span {
    int first, band, globals, gathered;  // first band tile, band tiles, gathered keys and their tiles
    int lo, hi;                          // positions of the first and the last row
};

template <int ROWS, int TILE>
__device__ __forceinline__ Span span_of(const AttnParams& p, const Globals& g, const Request& r, int q_tile) {
    Span s;
    const int n = p.per_group(r.rows);
    const int from = q_tile * ROWS, to = min(from + ROWS, r.rows) - 1;
    s.lo = r.len - n + p.per_group(from);
    s.hi = r.len - n + p.per_group(to);
    if (s.hi < 0) return {0, 0, 0, 0, s.lo, s.hi};
    int lo = max(0, s.lo - p.window);
    s.globals = 0;
    if (p.num_globals > 0) {
        if (lo > 0) {
            const int at = lower_bound(g.at, p.num_globals, s.lo);
            if (at < p.num_globals && g.at[at] <= s.hi) lo = 0;  // a global row sees every key up to itself
        }
        lo &= ~(TILE - 1);
        s.globals = lower_bound(g.at, p.num_globals, lo);
    }
    s.first = lo / TILE;
    s.band = s.hi / TILE - s.first + 1;
    s.gathered = (s.globals + TILE - 1) / TILE;
    return s;
}

template <int ROWS, int TILE>
__device__ __forceinline__ Request request_of(const AttnParams& p, const Globals& g, int b) {
    Request r = {0, 0, 0, 0, 0};
    if (b >= p.batch) return r;
    const int q0 = min(max(p.cu[b], 0), p.rows), q1 = min(max(p.cu[b + 1], 0), p.rows);
    if (q1 <= q0) return r;
    const int cap = p.width * p.pool.page_blocks * kBlock;
    r.q0 = q0;
    r.len = min(max(p.kv_lens[b], 0), cap);
    r.rows = (q1 - q0) * p.group;
    r.q_tiles = (r.rows + ROWS - 1) / ROWS;
    Span s = span_of<ROWS, TILE>(p, g, r, r.q_tiles - 1);
    r.tiles = s.band + s.gathered;
    if (r.q_tiles > 1) {
        // any tile: its rows lie within so many tokens, so its band within so many tiles; whole
        // when one of the new tokens is global
        const int tokens = (ROWS - 2) / p.group + 2;
        int band = (int)min((long long)(p.window + tokens - 1) / TILE + 2, (long long)r.len / TILE + 1);
        const int first = r.len - (q1 - q0);
        const int at = lower_bound(g.at, p.num_globals, first);
        if (at < p.num_globals && g.at[at] < r.len) band = r.len / TILE + 1;
        r.tiles = band + (lower_bound(g.at, p.num_globals, max(0, r.len - p.window)) + TILE - 1) / TILE;
    }
    r.tiles = max(r.tiles, 1);
    return r;
}

// a / b; the line of all but enormous calls fits 32 bits, whose division takes a fraction of the time.
__device__ __forceinline__ long long divide(long long a, int b) {
    return (a >> 32) == 0 ? (long long)((uint32_t)a / (uint32_t)b) : a / b;
}

__device__ __forceinline__ long long divide64(long long a, long long b) {
    return ((a | b) >> 32) == 0 ? (long long)((uint32_t)a / (uint32_t)b) : a / b;
}

__device__ __forceinline__ long long line_of(const AttnParams& p, const Request& r) {
    return (long long)r.q_tiles * p.pool.kv_heads * r.tiles;
}

// Block-wide: the sum of a value over the threads, and each thread's exclusive prefix.
template <int THREADS>
__device__ __forceinline__ long long block_scan(long long v, long long* scratch, long long* before) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long inc = v;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const long long u = __shfl_up_sync(kAll, inc, o);
        if (lane >= o) inc += u;
    }
    if (lane == 31) scratch[warp] = inc;
    __syncthreads();
    long long all = 0, mine = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
        if (w == warp) mine = all;
        all += scratch[w];
    }
    __syncthreads();
    *before = mine + inc - v;
    return all;
}

struct Place {
    int b;             // request; p.batch: none
    long long start;   // its first tile on the line
    Request r;
};

// The request that holds position `at` of the line, searched from `from` on, whose own part of the
// line begins at `start`.  `at` lies on the line.
template <int ROWS, int TILE, int THREADS>
__device__ __forceinline__ Place locate(const AttnParams& p, const Globals& g, int from, long long start, long long at,
                                        long long* scratch, Place* found) {
    for (int b0 = from; b0 < p.batch; b0 += THREADS) {
        const Request mine = request_of<ROWS, TILE>(p, g, b0 + (int)threadIdx.x);
        const long long line = line_of(p, mine);
        long long before;
        const long long all = block_scan<THREADS>(line, scratch, &before);
        if (at < start + all) {
            if (start + before <= at && at < start + before + line)
                *found = {b0 + (int)threadIdx.x, start + before, mine};
            __syncthreads();
            const Place r = *found;
            __syncthreads();
            return r;
        }
        start += all;
    }
    return {p.batch, start, {0, 0, 0, 0, 1}};
}

// A CTA's share [at, end) of the line, and where it begins.  One pass over the lengths where a
// thread holds one request, else one for the total and one for the place.
struct Share {
    long long per, at, end;
    Place here;
};

template <int ROWS, int TILE, int THREADS>
__device__ __forceinline__ Share share_of(const AttnParams& p, const Globals& g, long long* scratch, Place* found) {
    Share s;
    Request mine = {0, 0, 0, 0, 0};
    long long line = 0, before;
    for (int b = threadIdx.x; b < p.batch; b += THREADS) {
        mine = request_of<ROWS, TILE>(p, g, b);
        line += line_of(p, mine);
    }
    const long long all = block_scan<THREADS>(line, scratch, &before);
    s.per = divide(all + gridDim.x - 1, gridDim.x);
    if (p.split) s.per = max(s.per, (long long)p.min_tiles);
    s.at = s.per * blockIdx.x;
    s.end = min(s.at + s.per, all);
    s.here.b = p.batch;
    if (s.at >= s.end) return s;
    if (p.batch <= THREADS) {
        if (before <= s.at && s.at < before + line) *found = {(int)threadIdx.x, before, mine};
        __syncthreads();
        s.here = *found;
        __syncthreads();
    } else {
        s.here = locate<ROWS, TILE, THREADS>(p, g, 0, 0, s.at, scratch, found);
    }
    return s;
}

// Launch with programmatic stream serialisation: the kernel may be set up while the one before it in
// the stream drains.  Every CTA of a kernel launched so calls griddep_wait before it touches memory and
// before it returns, so the order of the stream's effects is unchanged.  LCA_PDL=0 in the environment launches in plain order.
template <typename... K, typename... A>
inline cudaError_t launch_early(void (*kernel)(K...), dim3 grid, unsigned block, size_t smem, cudaStream_t stream,
                                A&&... args) {
    static const bool on = [] {
        const char* e = getenv("LCA_PDL");
        return !(e != nullptr && e[0] == '0');
    }();
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = on ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, std::forward<A>(args)...);
}

// Dynamic shared memory beyond 48 KB for a kernel, asked for once per device.
template <typename F>
inline cudaError_t allow_smem(F* kernel, int bytes, std::atomic<unsigned long long>& done) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const unsigned long long bit = 1ull << (dev & 63);
    if (done.load(std::memory_order_acquire) & bit) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
    return e;
}

__device__ __forceinline__ void store_out(const AttnParams& p, int out_dtype, long long at, const float (&v)[4]) {
    if (out_dtype == LCA_DTYPE_F32) {
        *reinterpret_cast<float4*>(static_cast<float*>(p.out) + at) = make_float4(v[0], v[1], v[2], v[3]);
    } else if (out_dtype == LCA_DTYPE_F16) {
        const __half2 a = __floats2half2_rn(v[0], v[1]), b = __floats2half2_rn(v[2], v[3]);
        *reinterpret_cast<uint2*>(static_cast<__half*>(p.out) + at) =
            make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    } else {
        const __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
        *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.out) + at) =
            make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    }
}

}  // namespace kv4
}  // namespace lca
