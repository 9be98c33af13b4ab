// kv4_attention.cu -- causal sliding-window + global-token attention of new tokens over the paged
// 4-bit KV cache (format in kv4.h).
//
// With c a code, z the zero point and s the scale of its row (sk for K, sv for V), a request of
// `len` cached tokens whose last n are the new ones has its query row i at position
// p = len - n + i and computes, over the keys j <= p with p - j <= window, or j or p global,
//
//   x_j = scale * sk_j * sum_d q_d (ck_jd - zk_j),   O_d = sum_j e^(x_j - m) sv_j (cv_jd - zv_j) / l.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kv4.h"
#include "sm100_ptx.cuh"

namespace lca {
namespace kv4 {
namespace {

__device__ __forceinline__ float load_f(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ float load_f(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void store_f(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_f(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void store_f(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

__device__ __forceinline__ int lower_bound(const int32_t* a, int n, int v) {
    int lo = 0;
    while (lo < n) {
        const int mid = (lo + n) >> 1;
        if (a[mid] < v) lo = mid + 1; else n = mid;
    }
    return lo;
}

// One warp per (query row, head): a lane per key for the scores, then d / 32 elements a lane
// for the product with V.
template <int D, typename T, typename O>
__global__ void __launch_bounds__(128) kv4_attention_rows(const AttnParams p, const __grid_constant__ Globals g) {
    __shared__ float s_q[4][D];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long item = (long long)blockIdx.x * 4 + warp;
    if (item >= (long long)p.rows * p.heads) return;
    const int r = (int)(item / p.heads), head = (int)(item - (long long)r * p.heads), kv_head = head / p.group;
    if (r >= p.cu[p.batch] || r < p.cu[0]) return;  // rows outside the requests stay as they were
    int b = 0, hi = p.batch;
    while (b < hi) {
        const int mid = (b + hi) >> 1;
        if (p.cu[mid + 1] > r) hi = mid; else b = mid + 1;
    }
    const long long cap = min((long long)p.width * p.pool.page_blocks * kBlock, 0x7fffffffll);
    const int len = (int)min((long long)max(p.kv_lens[b], 0), cap);
    const int pos = len - (p.cu[b + 1] - r);
    for (int i = lane; i < D; i += 32) s_q[warp][i] = load_f(static_cast<const T*>(p.q) + r * p.q_token + head * p.q_head + i);
    __syncwarp();
    int lo = max(0, pos - p.window);
    const int at = lower_bound(g.at, p.num_globals, pos);
    if (at < p.num_globals && g.at[at] == pos) lo = 0;
    const int before = lower_bound(g.at, p.num_globals, lo);
    const int keys = pos < 0 ? 0 : before + pos + 1 - lo;
    float m = -INFINITY, l = 0.f, acc[D / 32] = {};
    for (int k0 = 0; k0 < keys; k0 += 32) {
        const int k = k0 + lane;
        float x = -INFINITY, sv = 0.f;
        const uint8_t* vrow = nullptr;
        int zv = 0;
        if (k < keys) {
            const int j = k < before ? g.at[k] : lo + k - before;
            const int blk = j / kBlock, row = j % kBlock;
            const int page = p.table[(long long)b * p.width + blk / p.pool.page_blocks];
            if (page >= 0 && page < p.pool.pages) {
                const uint8_t* block = p.pool.data + (((long long)page * p.pool.kv_heads + kv_head) * p.pool.page_blocks +
                                                      blk % p.pool.page_blocks) * block_bytes(D);
                const uint32_t wk = *reinterpret_cast<const uint32_t*>(block + k_words_at(D) + 4 * row);
                const uint32_t wv = *reinterpret_cast<const uint32_t*>(block + v_words_at(D) + 4 * row);
                const uint32_t* codes = reinterpret_cast<const uint32_t*>(block + row * row_bytes(D));
                const int zk = wk & 15u;
                float dot = 0.f;
                for (int i = 0; i < D / 8; ++i) {
                    const uint32_t c = codes[i];
                    for (int e = 0; e < 8; ++e) dot += s_q[warp][8 * i + e] * (float)((int)((c >> (4 * e)) & 15u) - zk);
                }
                x = dot * __uint_as_float(wk & ~15u) * p.scale;
                sv = __uint_as_float(wv & ~15u);
                zv = wv & 15u;
                vrow = block + v_codes_at(D) + row * row_bytes(D);
            }
        }
        float top = x;
        for (int o = 16; o > 0; o /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float m1 = fmaxf(m, top);
        const float ref = m1 == -INFINITY ? 0.f : m1;
        const float f = expf(m - ref);
        m = m1;
        const float e = vrow != nullptr ? expf(x - ref) : 0.f;
        l = l * f + e;
        for (int i = 0; i < D / 32; ++i) acc[i] *= f;
        for (int t = 0; t < 32; ++t) {
            const uint8_t* v = reinterpret_cast<const uint8_t*>(__shfl_sync(0xffffffffu, (unsigned long long)vrow, t));
            if (v == nullptr) continue;
            const float w = __shfl_sync(0xffffffffu, e * sv, t);
            const int z = __shfl_sync(0xffffffffu, zv, t);
            for (int i = 0; i < D / 32; ++i) {
                const int el = lane + 32 * i;
                const uint32_t c = (v[el / 2] >> (4 * (el & 1))) & 15u;
                acc[i] += w * (float)((int)c - z);
            }
        }
    }
    for (int o = 16; o > 0; o /= 2) l += __shfl_xor_sync(0xffffffffu, l, o);
    O* out = static_cast<O*>(p.out) + ((long long)r * p.heads + head) * D;
    for (int i = 0; i < D / 32; ++i) store_f(out + lane + 32 * i, l == 0.f ? 0.f : acc[i] / l);
    if (p.lse != nullptr && lane == 0) p.lse[(long long)head * p.rows + r] = l == 0.f ? -INFINITY : m + logf(l);
}

template <int D, typename T, typename O>
void attention_of(const AttnParams& p, const Globals& g, cudaStream_t stream) {
    const long long items = (long long)p.rows * p.heads;
    kv4_attention_rows<D, T, O><<<(unsigned)((items + 3) / 4), 128, 0, stream>>>(p, g);
}

template <int D, typename T>
void attention_out(int out_dtype, const AttnParams& p, const Globals& g, cudaStream_t stream) {
    if (out_dtype == LCA_DTYPE_F32)
        attention_of<D, T, float>(p, g, stream);
    else if (out_dtype == LCA_DTYPE_F16)
        attention_of<D, T, __half>(p, g, stream);
    else
        attention_of<D, T, __nv_bfloat16>(p, g, stream);
}

}  // namespace

cudaError_t launch_attention(int d, int dtype, int out_dtype, const AttnParams& p, const Globals& g,
                             cudaStream_t stream) {
    if (d == 64)
        dtype == LCA_DTYPE_F16 ? attention_out<64, __half>(out_dtype, p, g, stream)
                               : attention_out<64, __nv_bfloat16>(out_dtype, p, g, stream);
    else
        dtype == LCA_DTYPE_F16 ? attention_out<128, __half>(out_dtype, p, g, stream)
                               : attention_out<128, __nv_bfloat16>(out_dtype, p, g, stream);
    return cudaGetLastError();
}

}  // namespace kv4
}  // namespace lca
