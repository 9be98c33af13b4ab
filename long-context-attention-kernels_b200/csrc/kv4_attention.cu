// kv4_attention.cu -- causal sliding-window + global-token attention of new tokens over the paged
// 4-bit KV cache (format in kv4.h).
//
// With c a code, z the zero point and s the scale of its row (sk for K, sv for V), a request of
// `len` cached tokens whose last n are the new ones has its query row i at position
// p = len - n + i and computes, over the keys j <= p with p - j <= window, or j or p global,
//
//   x_j = scale * sk_j * sum_d q_d (ck_jd - zk_j),   O_d = sum_j e^(x_j - m) sv_j (cv_jd - zv_j) / l.
//
// The integers c - z are exact in fp16, so both products run on the tensor cores over them
// (mma.sync m16n8k16, keys by queries and elements by queries, fp32 sums) and the scales stay in
// fp32, outside the products: sk multiplies a finished score, sv the weight of its key.  For bf16
// outputs the scores take the codes unconverted: bits 0 .. 3 of an fp16 that is otherwise 0 are the
// subnormal c 2^-24, bits 4 .. 7 are c 2^-20, both exact operands, and zk_j sum_d q_d is taken off the sum.
// (That rounds to 2^-24 of sum |q_d| c_jd rather than of sum |q_d (c_jd - zk_j)|, which is too
// coarse for fp32 outputs; done to V, it would turn elements that are exactly 0 into such a
// remainder.)
#include <algorithm>

#include "kv4_attention.cuh"

namespace lca {
namespace kv4 {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kWholeKeys = 1536; // items of up to this many keys are not split
constexpr int kChunkFrom = 64;   // mean rows a request from which the tcgen05 kernel takes the call (both: plan_attention)
constexpr int kSms = 148;
constexpr int kCtas64 = 6;

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                     ptx::smem_u32(dst)),
                 "l"(src), "r"(bytes), "r"(ptx::smem_u32(bar))
                 : "memory");
}

__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Two codes of a word as fp16 subnormals: nibbles 0 and 4 (k = 0), 1 and 5 (16 times larger), 2 and 6, 3 and 7 (16
// times larger).
__device__ __forceinline__ uint32_t codes_raw(uint32_t w, int k) {
    const uint32_t v = k >= 2 ? w >> 8 : w;
    return v & ((k & 1) ? 0x00f000f0u : 0x000f000fu);
}

__device__ __forceinline__ float zero_of(uint32_t word) {  // 2^23 + z less 2^23
    return __uint_as_float((word & 15u) | 0x4b000000u) - 8388608.f;
}

__device__ __forceinline__ uint32_t transpose8(uint32_t a) {
    uint32_t d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}

// Resident CTAs of the streaming kernel on an SM: what its registers and its ring allow.
constexpr int ctas_per_sm(int d, int rows, int keys) {
    return rows == 8 ? (keys == 64 ? 3 : (d == 64 ? kCtas64 : 4)) : (rows == 16 ? 3 : 2);
}

// KB_: blocks of 16 keys per tile, one warp's step.
template <int D, int NT, int KB_>
struct Cfg {
    static constexpr int ROWS = 8 * NT;
    static constexpr int KB = KB_, TILE = 16 * KB, STAGES = KB == 2 ? 3 : 2;  // tiles in flight per warp
    static constexpr int STAGE = KB * block_bytes(D);
    static constexpr int RING = kWarps * STAGES * STAGE;
    static constexpr int PITCH = D + 4;  // floats of one row in the merge buffer
    static constexpr int MERGE = kWarps * ROWS * (PITCH + 2) * 4;
    static constexpr int MAIN = RING > MERGE ? RING : MERGE;
    static constexpr int SMEM = MAIN + kWarps * STAGES * 16;  // and the ring's barriers and key masks
};

// Position of slot s of a block in the products: the codes of slots 2t and 2t + 1 (V) and of slots
// g (K) are then read from shared memory with the fewest conflicts that a plain layout allows.
__device__ __forceinline__ int slot_row(int s) { return s ^ ((s >> 1) & 1); }

// One warp streams tiles of 64 (or 32) keys through its own ring of bulk copies and keeps the running
// softmax of 8 * NT query rows; the four warps of a CTA take the tiles of a segment in turn and
// merge at its end.  Per tile: scores S^T = K Q^T (keys are the 16 rows of the product, queries
// its 8 columns), weights, then O^T += V^T P^T.  The score fragment of a thread holds two
// queries of a key; transposed 8 x 8 it is the second product's operand.
//
// The weights w = p sv enter the second product as fp16 whatever the sizes of V, moved to the upper part of
// its range (kv4_attention.cuh, kHead); with an output finer than bf16 the remainder w - fp16(w) goes through
// a second product.
template <int D, int NT, int KB_, bool SPLIT_W>
__global__ void __launch_bounds__(kThreads, ctas_per_sm(D, 8 * NT, 16 * KB_))
    kv4_attention(const AttnParams p, const __grid_constant__ Globals g) {
    using C = Cfg<D, NT, KB_>;
    constexpr int STEPS = D / 16;  // products over d of a score, and 16-element tiles of O
    constexpr bool RAW_K = !SPLIT_W;  // scores over the codes as they are
    extern __shared__ __align__(128) uint8_t smem[];
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::MAIN);
    uint64_t* masks = bars + kWarps * C::STAGES;
    __shared__ long long scratch[kWarps];
    __shared__ Place found;

    const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31, gq = lane >> 2, t = lane & 3;
    const uint32_t pair_order = (t & 1) ? 0x1054u : 0x5410u;
    uint8_t* ring = smem + warp * C::STAGES * C::STAGE;
    uint64_t* bar = bars + warp * C::STAGES;
    uint64_t* mask = masks + warp * C::STAGES;  // keys of a tile that are there
    if (threadIdx.x < kWarps * C::STAGES) {
        ptx::mbar_init(&bars[threadIdx.x], 1);
        ptx::fence_mbar_init();
    }
    ptx::griddep_wait();

    const Share share = share_of<C::ROWS, C::TILE, kThreads>(p, g, scratch, &found);
    if (p.cuts != nullptr && threadIdx.x == 0) p.cuts[blockIdx.x].end = 0;  // until it cuts one off
    if (share.at >= share.end) return;
    const long long end = share.end;
    long long at = share.at;
    Place here = share.here;
    Request r = here.r;
    // the next slot of the ring to fill, and the next to empty with its phase
    int fill = 0, drain = 0, phase = 0;
    bool ok = true;

    while (here.b < p.batch) {
        const long long in = at - here.start;
        int item = (int)divide(in, r.tiles);
        int t0 = (int)(in - (long long)item * r.tiles), t1 = r.tiles;
        if (p.split) {
            t1 = (int)min((long long)r.tiles, t0 + (end - at));
        } else if (t0 > 0) {  // whole items only: this one belongs to the CTA before
            ++item;
            t0 = 0;
            at = here.start + (long long)item * r.tiles;
        }
        if (at >= end) break;
        const bool in_request = item < r.q_tiles * p.pool.kv_heads;
        if (in_request) {
            const int head = item / r.q_tiles, q_tile = item - head * r.q_tiles;
            Span span = span_of<C::ROWS, C::TILE>(p, g, r, q_tile);
            span.first = uniform(span.first), span.band = uniform(span.band);
            span.lo = uniform(span.lo), span.hi = uniform(span.hi);
            const int tiles = min(t1, span.band + span.gathered);
            const int mine = uniform(max(0, (tiles - t0 - warp + kWarps - 1) / kWarps)), first_tile = uniform(t0) + warp;
            const int32_t* table = p.table + (long long)here.b * p.width;

            // ---- loads: tile t0 + warp + 4 i of the item into the ring
            // Where the next tiles of this warp lie, a lane per block: index of the block in the pool (a
            // pool of 2^31 blocks would be 2 TB), -1 where there is none.  Fetched half of them ahead, so
            // that neither the table's latency nor the divisions are paid per tile.
            constexpr int KB = C::KB, AHEAD = 32 / KB;
            int where = -1, where_next = -1;
            auto fetch = [&](int i0) {
                const int i = i0 + lane / KB, tile = first_tile + kWarps * i, block = KB * (span.first + tile) + lane % KB;
                if (i >= mine || tile >= span.band || block > span.hi / kBlock) return -1;
                const int page_at = p.pool.per_page(block), page = table[page_at];
                if ((unsigned)page >= (unsigned)p.pool.pages) return -1;
                return (page * p.pool.kv_heads + head) * p.pool.page_blocks + block - page_at * p.pool.page_blocks;
            };
            auto issue = [&](int i) {
                if (i % AHEAD == 0) {
                    where = i == 0 ? fetch(0) : where_next;
                } else if (i % AHEAD == AHEAD / 2) {
                    where_next = fetch(i - AHEAD / 2 + AHEAD);
                }
                const int slot = fill;
                fill = fill + 1 == C::STAGES ? 0 : fill + 1;
                uint8_t* dst = ring + slot * C::STAGE;
                const int tile = first_tile + kWarps * i;
                if (tile < span.band) {
                    int at[KB];
#pragma unroll
                    for (int k = 0; k < KB; ++k) at[k] = __shfl_sync(kAll, where, KB * (i % AHEAD) + k);
                    if (lane == 0) {
                        bool run = at[0] >= 0;
                        uint64_t have = 0;
                        int count = 0;
#pragma unroll
                        for (int k = 0; k < KB; ++k) {
                            run &= at[k] == at[0] + k;
                            have |= at[k] >= 0 ? 0xffffull << (16 * k) : 0ull;
                            count += at[k] >= 0;
                        }
                        mask[slot] = have;
                        ptx::mbar_arrive_expect_tx(&bar[slot], count * block_bytes(D));
                        if (run) {  // blocks of one page follow one another
                            bulk_load(dst, p.pool.data + (long long)at[0] * block_bytes(D), C::STAGE, &bar[slot]);
                        } else {
#pragma unroll
                            for (int k = 0; k < KB; ++k)
                                if (at[k] >= 0)
                                    bulk_load(dst + k * block_bytes(D), p.pool.data + (long long)at[k] * block_bytes(D),
                                              block_bytes(D), &bar[slot]);
                        }
                    }
                } else {  // gathered global tokens, a lane for every 32nd
                    const uint8_t* src[KB / 2];
                    int row[KB / 2];
                    uint64_t have = 0;
#pragma unroll
                    for (int e = 0; e < KB / 2; ++e) {
                        const int k = (tile - span.band) * C::TILE + 32 * e + lane;
                        src[e] = nullptr;
                        row[e] = 0;
                        if (k < span.globals) {
                            const int pos = g.at[k], block = pos / kBlock, page_at = p.pool.per_page(block);
                            row[e] = pos % kBlock;
                            const int page = table[page_at];
                            if ((unsigned)page < (unsigned)p.pool.pages)
                                src[e] = p.pool.data + (long long)((page * p.pool.kv_heads + head) * p.pool.page_blocks + block -
                                                                   page_at * p.pool.page_blocks) * block_bytes(D);
                        }
                        have |= (uint64_t)__ballot_sync(kAll, src[e] != nullptr) << (32 * e);
                    }
                    uint8_t* to = dst + (lane >> 4) * block_bytes(D);
                    const int to_row = lane & 15;
#pragma unroll
                    for (int e = 0; e < KB / 2; ++e) {
                        if (src[e] == nullptr) continue;
                        uint8_t* words = to + 2 * e * block_bytes(D) + 4 * to_row;
                        *reinterpret_cast<uint32_t*>(words + k_words_at(D)) =
                            *reinterpret_cast<const uint32_t*>(src[e] + k_words_at(D) + 4 * row[e]);
                        *reinterpret_cast<uint32_t*>(words + v_words_at(D)) =
                            *reinterpret_cast<const uint32_t*>(src[e] + v_words_at(D) + 4 * row[e]);
                    }
                    ptx::fence_proxy_async_smem();  // a later copy may land on these words
                    if (lane == 0) {
                        mask[slot] = have;
                        ptx::mbar_arrive_expect_tx(&bar[slot], __popcll(have) * D);
                    }
                    __syncwarp();
#pragma unroll
                    for (int e = 0; e < KB / 2; ++e) {
                        if (src[e] == nullptr) continue;
                        uint8_t* codes = to + 2 * e * block_bytes(D) + to_row * row_bytes(D);
                        bulk_load(codes, src[e] + row[e] * row_bytes(D), row_bytes(D), &bar[slot]);
                        bulk_load(codes + v_codes_at(D), src[e] + v_codes_at(D) + row[e] * row_bytes(D), row_bytes(D),
                                  &bar[slot]);
                    }
                }
                __syncwarp();
            };
            int issued = 0;
            if (ok)
                for (; issued < min(mine, C::STAGES); ++issued) issue(issued);

            // ---- queries: rows of the tile as the second operand, in the order of the K codes
            uint32_t q[NT][STEPS][2];
            float q_scale[NT][2], q_total[NT][2];  // of this thread's two columns
            int row_hi[NT][2], row_lo[NT][2];  // their positions and band starts
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const int row = q_tile * C::ROWS + 8 * nt + gq;
                uint32_t raw[D / 8];
                if (row < r.rows) {
                    const int token = p.per_group(row), of = row - token * p.group;
                    const uint4* src = reinterpret_cast<const uint4*>(
                        static_cast<const uint16_t*>(p.q) + (r.q0 + token) * p.q_token +
                        (long long)(head * p.group + of) * p.q_head + t * (D / 4));
#pragma unroll
                    for (int i = 0; i < D / 32; ++i) {
                        const uint4 v = src[i];
                        raw[4 * i] = v.x, raw[4 * i + 1] = v.y, raw[4 * i + 2] = v.z, raw[4 * i + 3] = v.w;
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < D / 8; ++i) raw[i] = 0;
                }
                // moved by a power of two that takes the row's largest element to [2^14, 2^15), where fp16 holds
                // every bit of elements down to 2^-25 of it (2^-21 of a quarter of them below)
                float mult = fabsf(p.scale) * kLog2e;
                uint32_t top = 0;
#pragma unroll
                for (int i = 0; i < D / 8; ++i) top = max(top, max(raw[i] & 0x7fffu, (raw[i] >> 16) & 0x7fffu));
                top = max(top, __shfl_xor_sync(kAll, top, 1));
                top = max(top, __shfl_xor_sync(kAll, top, 2));
                float total = 0.f;  // of the row's elements, as they enter the product
                {
                    const int e = p.bf16 ? max((int)(top >> 7) - 127, -100)  // above 2^-100; smaller rows score 0
                                         : max((int)(top >> 10) - 15, -14);
                    const float up = __uint_as_float((uint32_t)(14 - e + 127) << 23);
                    mult *= __uint_as_float((uint32_t)max(e - 14 + 127, 0) << 23);
                    if (p.scale < 0.f) mult = -mult;
#pragma unroll
                    for (int i = 0; i < D / 8; ++i) {
                        float2 x;
                        if (p.bf16)
                            x = make_float2(__uint_as_float(raw[i] << 16), __uint_as_float(raw[i] & 0xffff0000u));
                        else
                            x = __half22float2(*reinterpret_cast<const __half2*>(&raw[i]));
                        raw[i] = ptx::pack_f16x2(x.x * up, x.y * up);
                    }
                }
                // The factor of a score is positive and finite, so that it leaves the -inf of a masked
                // one alone: the scale's sign goes to the row, a factor of 0 makes it a row of zeros,
                // and a row that is not finite, or a scale that is not, a row of NaN.
                const bool finite = top < (p.bf16 ? 0x7f80u : 0x7c00u) && fabsf(mult) < INFINITY;
                const bool zero = fabsf(mult) < 1.17549435e-38f;
                const uint32_t flip = mult < 0.f ? 0x80008000u : 0u;
                mult = !finite || zero ? 1.f : fabsf(mult);
#pragma unroll
                for (int i = 0; i < D / 8; ++i) {
                    raw[i] ^= flip;
                    if (zero) raw[i] = 0;
                    if (!finite) raw[i] = 0x7e007e00u;
                    const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&raw[i]));
                    total += x.x + x.y;
                }
                if (RAW_K) mult *= 16777216.f;  // the codes are 2^-24 of themselves
#pragma unroll
                for (int w = 0; w < D / 32; ++w) {  // elements 8w .. 8w + 7 of this thread's chunk
                    q[nt][2 * w][0] = __byte_perm(raw[4 * w], raw[4 * w + 2], 0x5410);
                    q[nt][2 * w][1] = __byte_perm(raw[4 * w], raw[4 * w + 2], 0x7632);
                    q[nt][2 * w + 1][0] = __byte_perm(raw[4 * w + 1], raw[4 * w + 3], 0x5410);
                    q[nt][2 * w + 1][1] = __byte_perm(raw[4 * w + 1], raw[4 * w + 3], 0x7632);
                    if (RAW_K) {  // against codes that are 16 times larger
                        q[nt][2 * w][1] = hmul2(q[nt][2 * w][1], 0x2c002c00u);
                        q[nt][2 * w + 1][1] = hmul2(q[nt][2 * w + 1][1], 0x2c002c00u);
                    }
                }
                total += __shfl_xor_sync(kAll, total, 1);
                total += __shfl_xor_sync(kAll, total, 2);
                total *= 1.f / 16777216.f;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    q_scale[nt][e] = __shfl_sync(kAll, mult, 4 * (2 * t + e));
                    q_total[nt][e] = __shfl_sync(kAll, total, 4 * (2 * t + e));
                    const int col = q_tile * C::ROWS + 8 * nt + 2 * t + e;
                    const int pos = col < r.rows ? r.len - p.per_group(r.rows) + p.per_group(col) : -1;
                    row_hi[nt][e] = pos;
                    row_lo[nt][e] = max(0, pos - p.window);
                    if (p.num_globals > 0 && span.first == 0) {
                        const int k = lower_bound(g.at, p.num_globals, pos);
                        if (k < p.num_globals && g.at[k] == pos) row_lo[nt][e] = 0;
                    }
                }
            }

            float o[NT][STEPS][4], top[NT][2], sum[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                top[nt][0] = top[nt][1] = -INFINITY;
                sum[nt][0] = sum[nt][1] = 0.f;
#pragma unroll
                for (int i = 0; i < STEPS; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
            }

#pragma unroll 1
            for (int i = 0; i < issued; ++i) {
                const int slot = drain;
                if (!ptx::mbar_wait(&bar[slot], phase, nullptr, p.err_word, LCA_DEVERR_TIMEOUT_CACHE,
                                    p.wait_ns))
                    ok = false;
                drain = drain + 1 == C::STAGES ? 0 : drain + 1;
                phase ^= drain == 0;
                ok = __all_sync(kAll, ok);
                if (!ok) continue;  // results are invalid; the copies still in flight are waited for
                const uint8_t* stage = ring + slot * C::STAGE;
                const int tile = first_tile + kWarps * i;
                const int key0 = (span.first + tile) * C::TILE;
                const uint64_t have = mask[slot];
                const int row0 = slot_row(gq);

                // ---- scores
                float s[KB][NT][4];
                float sk[2 * KB], sv[2 * KB], zk[2 * KB];
#pragma unroll
                for (int m = 0; m < KB; ++m) {
                    const uint8_t* block = stage + m * block_bytes(D);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) s[m][nt][0] = s[m][nt][1] = s[m][nt][2] = s[m][nt][3] = 0.f;
                    const uint32_t w0 = *reinterpret_cast<const uint32_t*>(block + k_words_at(D) + 4 * row0);
                    const uint32_t w1 = *reinterpret_cast<const uint32_t*>(block + k_words_at(D) + 4 * row0 + 32);
                    sk[2 * m] = __uint_as_float(w0 & ~15u);
                    sk[2 * m + 1] = __uint_as_float(w1 & ~15u);
                    const uint32_t w2 = *reinterpret_cast<const uint32_t*>(block + v_words_at(D) + 4 * row0);
                    const uint32_t w3 = *reinterpret_cast<const uint32_t*>(block + v_words_at(D) + 4 * row0 + 32);
                    sv[2 * m] = __uint_as_float(w2 & ~15u);
                    sv[2 * m + 1] = __uint_as_float(w3 & ~15u);
                    zk[2 * m] = zero_of(w0);
                    zk[2 * m + 1] = zero_of(w1);
                    const Zero z0 = zero_pair((w0 & 15u) * 0x10001u), z1 = zero_pair((w1 & 15u) * 0x10001u);
                    uint32_t c0[D / 32], c1[D / 32];
                    const uint8_t* at0 = block + row0 * row_bytes(D) + t * (D / 8);
                    const uint8_t* at1 = at0 + 8 * row_bytes(D);
                    if (D == 128) {
                        *reinterpret_cast<uint4*>(c0) = *reinterpret_cast<const uint4*>(at0);
                        *reinterpret_cast<uint4*>(c1) = *reinterpret_cast<const uint4*>(at1);
                    } else {
                        *reinterpret_cast<uint2*>(c0) = *reinterpret_cast<const uint2*>(at0);
                        *reinterpret_cast<uint2*>(c1) = *reinterpret_cast<const uint2*>(at1);
                    }
#pragma unroll
                    for (int w = 0; w < D / 32; ++w) {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const uint32_t a0 = RAW_K ? codes_raw(c0[w], 2 * h) : codes_pair(c0[w], 2 * h, z0);
                            const uint32_t a1 = RAW_K ? codes_raw(c1[w], 2 * h) : codes_pair(c1[w], 2 * h, z1);
                            const uint32_t a2 = RAW_K ? codes_raw(c0[w], 2 * h + 1) : codes_pair(c0[w], 2 * h + 1, z0);
                            const uint32_t a3 = RAW_K ? codes_raw(c1[w], 2 * h + 1) : codes_pair(c1[w], 2 * h + 1, z1);
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt)
                                mma(s[m][nt], a0, a1, a2, a3, q[nt][2 * w + h][0], q[nt][2 * w + h][1]);
                        }
                    }
                }

                // ---- visibility: nothing to do where the whole tile is visible to every row
                const bool band = tile < span.band;
                const bool full = __all_sync(kAll, have == (KB == 4 ? ~0ull : 0xffffffffull)) &&
                                  (!band || (key0 + C::TILE - 1 <= span.lo && key0 >= span.hi - p.window));
                uint32_t seen[NT];  // bit c = 4 m + 2 (second row) + column
                if (!full) {
                    uint64_t glob = 0;  // global keys of the tile, which rows outside whose band they lie see
                    if (band && p.num_globals > 0) {
#pragma unroll
                        for (int e = 0; e < KB / 2; ++e) {
                            const int key = key0 + 32 * e + lane, k = lower_bound(g.at, p.num_globals, key);
                            glob |= (uint64_t)__ballot_sync(kAll, k < p.num_globals && g.at[k] == key) << (32 * e);
                        }
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        seen[nt] = 0;
#pragma unroll
                        for (int c = 0; c < 4 * KB; ++c) {
                            const int k = 16 * (c >> 2) + 8 * ((c >> 1) & 1) + row0, e = c & 1;
                            const bool there = (have >> k) & 1;
                            const int j = key0 + k;
                            const bool vis = there && (band ? j <= row_hi[nt][e] && (j >= row_lo[nt][e] || ((glob >> k) & 1))
                                                            : row_hi[nt][e] >= 0);
                            seen[nt] |= (uint32_t)vis << c;
                        }
                    }
                }

                // ---- softmax
                float lam[2 * KB];
#pragma unroll
                for (int c = 0; c < 2 * KB; ++c) lam[c] = fmaxf(lg2(fabsf(sv[c])), kLeast);
                bool raise = false;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                    for (int c = 0; c < 4 * KB; ++c) {
                        float& x = s[c >> 2][nt][c & 3];
                        if (RAW_K) x -= zk[c >> 1] * q_total[nt][c & 1];
                        x *= sk[c >> 1];
                    }
                    if (!full) {
#pragma unroll
                        for (int c = 0; c < 4 * KB; ++c)
                            if (!((seen[nt] >> c) & 1)) s[c >> 2][nt][c & 3] = -INFINITY;
                    }
                }
                auto peaks = [&](int nt, int e) {  // of this thread's keys
                    float m = -INFINITY;
#pragma unroll
                    for (int k = 0; k < KB; ++k)
                        m = ptx::fmax3(m, s[k][nt][e] * q_scale[nt][e] + lam[2 * k],
                                       s[k][nt][2 + e] * q_scale[nt][e] + lam[2 * k + 1]);
                    return m;
                };
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) raise |= peaks(nt, 0) > top[nt][0] + kRise || peaks(nt, 1) > top[nt][1] + kRise;
                if (__any_sync(kAll, raise)) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        float f[2];
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            float to = peaks(nt, e);
#pragma unroll
                            for (int m = 4; m < 32; m *= 2) to = fmaxf(to, __shfl_xor_sync(kAll, to, m));
                            const bool rise = to > top[nt][e] + kRise;
                            to = rise ? to - kHead : top[nt][e];
                            const float half = rise ? ex2_half(top[nt][e] - to) : 1.f;
                            top[nt][e] = to;
                            sum[nt][e] = half * (half * sum[nt][e]);
                            f[e] = half * half;
                        }
#pragma unroll
                        for (int k = 0; k < STEPS; ++k) {
                            o[nt][k][0] *= f[0], o[nt][k][1] *= f[1];
                            o[nt][k][2] *= f[0], o[nt][k][3] *= f[1];
                        }
                    }
                }
                uint32_t w_hi[NT][2 * KB], w_lo[NT][2 * KB];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const float ref0 = top[nt][0] == -INFINITY ? 0.f : top[nt][0];
                    const float ref1 = top[nt][1] == -INFINITY ? 0.f : top[nt][1];
                    float w[4 * KB];
#pragma unroll
                    for (int c = 0; c < 2 * KB; ++c) {  // key row c of this thread, both columns
                        const float* x = &s[c >> 1][nt][2 * (c & 1)];
                        const float p0 = ptx::ex2(x[0] * q_scale[nt][0] - ref0), p1 = ptx::ex2(x[1] * q_scale[nt][1] - ref1);
                        sum[nt][0] += p0;
                        sum[nt][1] += p1;
                        w[2 * c] = p0 * sv[c];
                        w[2 * c + 1] = p1 * sv[c];
                    }
                    if (!full) {  // 0 also where the scale of a key that is not there is not finite
#pragma unroll
                        for (int c = 0; c < 4 * KB; ++c)
                            if (!((seen[nt] >> c) & 1)) w[c] = 0.f;
                    }
#pragma unroll
                    for (int c = 0; c < 2 * KB; ++c) {
                        const uint32_t hi = ptx::pack_f16x2(w[2 * c], w[2 * c + 1]);
                        w_hi[nt][c] = transpose8(hi);
                        if (SPLIT_W) {
                            const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&hi));
                            w_lo[nt][c] = transpose8(ptx::pack_f16x2(w[2 * c] - back.x, w[2 * c + 1] - back.y));
                        }
                    }
                }

                // ---- product with V
#pragma unroll
                for (int m = 0; m < KB; ++m) {
                    const uint8_t* block = stage + m * block_bytes(D);
                    const int r0 = slot_row(2 * t), r1 = slot_row(2 * t + 1);
                    // r0 and r1 are 2t and 2t + 1, in that order for an even t
                    const uint2 w01 = *reinterpret_cast<const uint2*>(block + v_words_at(D) + 8 * t);
                    const uint2 w23 = *reinterpret_cast<const uint2*>(block + v_words_at(D) + 8 * t + 32);
                    const Zero z01 = zero_pair(__byte_perm(w01.x, w01.y, pair_order) & 0x000f000fu);
                    const Zero z23 = zero_pair(__byte_perm(w23.x, w23.y, pair_order) & 0x000f000fu);
                    const uint8_t* codes = block + v_codes_at(D) + gq * (D / 16);
                    // [half of the m-tile's rows][low or high 16 bits of a word]
                    uint32_t a01[2][2], a23[2][2];
                    if (D == 128) {
                        const uint2 x0 = *reinterpret_cast<const uint2*>(codes + r0 * row_bytes(D));
                        const uint2 x1 = *reinterpret_cast<const uint2*>(codes + r1 * row_bytes(D));
                        const uint2 x2 = *reinterpret_cast<const uint2*>(codes + (r0 + 8) * row_bytes(D));
                        const uint2 x3 = *reinterpret_cast<const uint2*>(codes + (r1 + 8) * row_bytes(D));
                        a01[0][0] = __byte_perm(x0.x, x1.x, 0x5410), a01[0][1] = __byte_perm(x0.x, x1.x, 0x7632);
                        a01[1][0] = __byte_perm(x0.y, x1.y, 0x5410), a01[1][1] = __byte_perm(x0.y, x1.y, 0x7632);
                        a23[0][0] = __byte_perm(x2.x, x3.x, 0x5410), a23[0][1] = __byte_perm(x2.x, x3.x, 0x7632);
                        a23[1][0] = __byte_perm(x2.y, x3.y, 0x5410), a23[1][1] = __byte_perm(x2.y, x3.y, 0x7632);
                    } else {
                        const uint32_t x0 = *reinterpret_cast<const uint32_t*>(codes + r0 * row_bytes(D));
                        const uint32_t x1 = *reinterpret_cast<const uint32_t*>(codes + r1 * row_bytes(D));
                        const uint32_t x2 = *reinterpret_cast<const uint32_t*>(codes + (r0 + 8) * row_bytes(D));
                        const uint32_t x3 = *reinterpret_cast<const uint32_t*>(codes + (r1 + 8) * row_bytes(D));
                        a01[0][0] = __byte_perm(x0, x1, 0x5410), a01[1][0] = __byte_perm(x0, x1, 0x7632);
                        a23[0][0] = __byte_perm(x2, x3, 0x5410), a23[1][0] = __byte_perm(x2, x3, 0x7632);
                        a01[0][1] = a01[1][1] = a23[0][1] = a23[1][1] = 0;
                    }
#pragma unroll
                    for (int k = 0; k < STEPS; ++k) {
                        const int part = k >> 2, nib = k & 3;
                        const uint32_t b0 = codes_pair(a01[0][part], nib, z01), b1 = codes_pair(a01[1][part], nib, z01);
                        const uint32_t b2 = codes_pair(a23[0][part], nib, z23), b3 = codes_pair(a23[1][part], nib, z23);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            mma(o[nt][k], b0, b1, b2, b3, w_hi[nt][2 * m], w_hi[nt][2 * m + 1]);
                            if (SPLIT_W) mma(o[nt][k], b0, b1, b2, b3, w_lo[nt][2 * m], w_lo[nt][2 * m + 1]);
                        }
                    }
                }
                __syncwarp();
                if (issued < mine) {
                    issue(issued);
                    ++issued;
                }
            }
            // ---- the four warps' parts of the segment
            __syncthreads();
            // The next kernel may be set up now.  Not earlier: its CTAs would take the places that are free
            // while this grid runs, which are not spread evenly, and keep them.
            if (at + (t1 - t0) >= end) ptx::griddep_launch();
            float* buf = reinterpret_cast<float*>(smem);
            float2* stats = reinterpret_cast<float2*>(buf + kWarps * C::ROWS * C::PITCH);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
#pragma unroll
                    for (int m = 4; m < 32; m *= 2) sum[nt][e] += __shfl_xor_sync(kAll, sum[nt][e], m);
                    const int row = warp * C::ROWS + 8 * nt + 2 * t + e;
                    if (gq == 0) stats[row] = make_float2(top[nt][e], sum[nt][e]);
                    float* to = buf + row * C::PITCH + gq * (D / 8);
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int k = 0; k < STEPS; k += 4)
                            *reinterpret_cast<float4*>(to + h * STEPS + k) =
                                make_float4(o[nt][k][2 * h + e], o[nt][k + 1][2 * h + e], o[nt][k + 2][2 * h + e],
                                            o[nt][k + 3][2 * h + e]);
                }
            }
            __syncthreads();
            const bool whole = t0 == 0 && t1 == r.tiles;
            const int part = (int)(2 * blockIdx.x) + (at != share.at);
            if (p.cuts != nullptr && t0 == 0 && t1 < r.tiles && threadIdx.x == 0)
                p.cuts[blockIdx.x] = {at + r.tiles, share.per, at != share.at, r.q0, r.rows, head, q_tile};
            for (int x = threadIdx.x; x < C::ROWS * (D / 4); x += kThreads) {
                const int row = x / (D / 4), d = 4 * (x - row * (D / 4));
                const int of = q_tile * C::ROWS + row;
                if (of >= r.rows) continue;
                float m = -INFINITY;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) m = fmaxf(m, stats[w * C::ROWS + row].x);
                const float ref = m == -INFINITY ? 0.f : m;
                float l = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int w = 0; w < kWarps; ++w) {
                    const float2 st = stats[w * C::ROWS + row];
                    const float half = ex2_half(st.x - ref), f = half * half;
                    l += half * (half * st.y);
                    const float4 a = *reinterpret_cast<const float4*>(buf + (w * C::ROWS + row) * C::PITCH + d);
                    v[0] += f * a.x, v[1] += f * a.y, v[2] += f * a.z, v[3] += f * a.w;
                }
                if (whole) {
                    const int token = p.per_group(of), h = head * p.group + of - token * p.group;
                    const float inv = l == 0.f ? 0.f : 1.f / l;
                    if (l == 0.f) v[0] = v[1] = v[2] = v[3] = 0.f;
                    v[0] *= inv, v[1] *= inv, v[2] *= inv, v[3] *= inv;
                    store_out(p, p.out_dtype, ((long long)(r.q0 + token) * p.heads + h) * D + d, v);
                    if (p.lse != nullptr && d == 0)
                        p.lse[(long long)h * p.rows + r.q0 + token] = lse_of(m, l);
                } else {
                    const long long to = (long long)part * C::ROWS + row;
                    *reinterpret_cast<float4*>(p.part_o + to * D + d) = make_float4(v[0], v[1], v[2], v[3]);
                    if (d == 0) p.part_ml[to] = make_float2(m, l);
                }
            }
            ptx::fence_proxy_async_smem();  // the next copies land where these values were
            __syncthreads();
        }
        at = p.split ? at + (t1 - t0) : at + r.tiles;
        if (!in_request) at = here.start + line_of(p, r);
        if (at >= end) break;
        if (at >= here.start + line_of(p, r)) {
            here = locate<C::ROWS, C::TILE, kThreads>(p, g, here.b + 1, here.start + line_of(p, r), at, scratch, &found);
            r = here.r;
        }
    }
}

// The parts of the items that several CTAs shared: one CTA per (item, row), a warp per eighth of the
// parts.  Parts are summed in the order of the line, so a call's result does not depend on timing.
// Where there are fewer items than CTAs of the attention, a CTA finds its item from the lengths; else it
// takes the item that its namesake cut.  Set up while the attention drains (programmatic launch), but every
// CTA waits for it first, also one that has nothing to merge: what follows in the stream is ordered behind
// this grid alone, which must not complete before the attention has.
constexpr int kMergeWarps = 8;

template <int D, int ROWS, int TILE>
__global__ void __launch_bounds__(32 * kMergeWarps) kv4_attention_merge(const AttnParams p, const __grid_constant__ Globals g) {
    constexpr int THREADS = 32 * kMergeWarps, PER = D / 32;
    __shared__ long long scratch[kMergeWarps];
    __shared__ Place found;
    __shared__ int found_item;
    __shared__ float s_m[kMergeWarps], s_l[kMergeWarps], s_o[kMergeWarps][D];
    const int id = blockIdx.x, row = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    ptx::griddep_wait();
    Cut cut = {};
    int c0 = id, c1;
    if (p.cuts != nullptr) {  // a CTA per CTA of the attention
        cut = p.cuts[id];
        if (cut.end == 0) return;
        c1 = (int)divide64(cut.end - 1, cut.per);
    } else {  // a CTA per item: few of them, so few lengths too
        if (threadIdx.x == 0) found.b = -1;
        long long line = 0, items = 0;
        for (int b0 = 0; b0 < p.batch; b0 += THREADS) {
            const Request r = request_of<ROWS, TILE>(p, g, b0 + (int)threadIdx.x);
            const long long mine = line_of(p, r), count = (long long)r.q_tiles * p.pool.kv_heads;
            long long before, items_before;
            const long long all = block_scan<THREADS>(mine, scratch, &before);
            const long long all_items = block_scan<THREADS>(count, scratch, &items_before);
            if (items + items_before <= id && id < items + items_before + count) {
                found = {b0 + (int)threadIdx.x, line + before, r};
                found_item = (int)(id - items - items_before);
            }
            line += all;
            items += all_items;
        }
        __syncthreads();
        if (found.b < 0) return;
        const Request r = found.r;
        const long long per = max(divide(line + p.ctas - 1, p.ctas), (long long)p.min_tiles);
        const long long s = found.start + (long long)found_item * r.tiles;
        c0 = (int)divide64(s, per);
        c1 = (int)divide64(s + r.tiles - 1, per);
        cut.slot = s > c0 * per;
        cut.q0 = r.q0;
        cut.rows = r.rows;
        cut.head = found_item / r.q_tiles;
        cut.q_tile = found_item - cut.head * r.q_tiles;
        if (c0 == c1) return;  // one CTA had it all and wrote the output
    }
    const int of = cut.q_tile * ROWS + row;
    if (of >= cut.rows) return;

    auto part_of = [&](int c) { return (2ll * c + (c == c0 ? cut.slot : 0)) * ROWS + row; };
    float m = -INFINITY, l = 0.f, o[PER] = {};
    for (int c = c0 + warp; c <= c1; c += kMergeWarps) m = fmaxf(m, p.part_ml[part_of(c)].x);
    const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll 4
    for (int c = c0 + warp; c <= c1; c += kMergeWarps) {
        const long long at = part_of(c);
        const float2 ml = p.part_ml[at];
        const float half = ex2_half(ml.x - ref), f = half * half;
        l += half * (half * ml.y);
        const float* src = p.part_o + at * D + lane * PER;
        if (PER == 4) {
            const float4 v = *reinterpret_cast<const float4*>(src);
            o[0] += f * v.x, o[1] += f * v.y, o[PER - 2] += f * v.z, o[PER - 1] += f * v.w;
        } else {
            const float2 v = *reinterpret_cast<const float2*>(src);
            o[0] += f * v.x, o[1] += f * v.y;
        }
    }
    if (lane == 0) s_m[warp] = m, s_l[warp] = l;
#pragma unroll
    for (int i = 0; i < PER; ++i) s_o[warp][lane * PER + i] = o[i];
    __syncthreads();
    if (threadIdx.x >= D / 4) return;
    float top = -INFINITY, sum = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kMergeWarps; ++w) top = fmaxf(top, s_m[w]);
    const float ref_top = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int w = 0; w < kMergeWarps; ++w) {
        const float half = ex2_half(s_m[w] - ref_top), f = half * half;
        sum += half * (half * s_l[w]);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] += f * s_o[w][4 * threadIdx.x + i];
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = sum == 0.f ? 0.f : v[i] * inv;
    const int token = p.per_group(of), h = cut.head * p.group + of - token * p.group;
    store_out(p, p.out_dtype, ((long long)(cut.q0 + token) * p.heads + h) * D + 4 * threadIdx.x, v);
    if (p.lse != nullptr && threadIdx.x == 0)
        p.lse[(long long)h * p.rows + cut.q0 + token] = lse_of(top, sum);
}

template <int D, int ROWS, int TILE>
cudaError_t merge_of(const AttnParams& p, const Globals& g, cudaStream_t stream) {
    return launch_early(kv4_attention_merge<D, ROWS, TILE>, dim3(p.cuts != nullptr ? p.ctas : (unsigned)p.items, ROWS), 32 * kMergeWarps, 0, stream, p, g);
}

template <int D, int NT, int KB, bool SPLIT_W>
cudaError_t attention_of(const AttnParams& p, const Globals& g, cudaStream_t stream) {
    const int smem = Cfg<D, NT, KB>::SMEM;
    static std::atomic<unsigned long long> done{0};
    cudaError_t e = allow_smem(kv4_attention<D, NT, KB, SPLIT_W>, smem, done);
    if (e != cudaSuccess) return e;
    e = launch_early(kv4_attention<D, NT, KB, SPLIT_W>, dim3(p.ctas), kThreads, smem, stream, p, g);
    return e != cudaSuccess || !p.split ? e : merge_of<D, 8 * NT, 16 * KB>(p, g, stream);
}

template <int D, int NT, int KB>
cudaError_t attention_tiles(const AttnParams& p, const Globals& g, cudaStream_t stream) {
    // bf16 is rounded more coarsely than the weights are
    return p.out_dtype != LCA_DTYPE_BF16 ? attention_of<D, NT, KB, true>(p, g, stream)
                                         : attention_of<D, NT, KB, false>(p, g, stream);
}

template <int D>
cudaError_t attention_rows(int tile_rows, int tile_keys, const AttnParams& p, const Globals& g, cudaStream_t stream) {
    if (tile_rows == 8)
        return tile_keys == 64 ? attention_tiles<D, 1, 4>(p, g, stream) : attention_tiles<D, 1, 2>(p, g, stream);
    if (tile_rows == 16) return attention_tiles<D, 2, 2>(p, g, stream);
    if (tile_rows == 32) return attention_tiles<D, 4, 2>(p, g, stream);
    const cudaError_t e = launch_chunk(D, p, g, stream);
    return e != cudaSuccess || !p.split ? e : merge_of<D, kChunkRows, kChunkKeys>(p, g, stream);
}

}  // namespace

// Rows of an item: as many groups of 8 as an average request has, so that a tile of keys is
// unpacked once for all of them, up to the 32 whose sums fit the registers of one warp; from
// kChunkFrom rows on, 256 rows on tcgen05.  Measured with 32 / 8 heads of 128 (one kernel | the other, us), 48, 64 and
// 96 rows a request over whole contexts of 16K to 32K: one request 62 | 63, 65 | 63, 83 | 66; 32 of them 899 | 1080,
// 911 | 1086, 1336 | 1095; with a window of 512, 32 requests of 32, 48 and 64 rows 34 | 49, 62 | 48, 65 | 49.
AttnPlan plan_attention(int64_t rows, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t batch, int64_t capacity,
                        int64_t window, int64_t num_globals) {
    AttnPlan a = {};
    if (rows <= 0 || batch <= 0) return a;
    const int64_t group = heads / kv_heads;
    const int64_t mean = (rows + batch - 1) / batch * group;
    const bool chunk = mean >= kChunkFrom;
    a.tile_rows = chunk ? kChunkRows : (mean <= 8 ? 8 : (mean <= 16 ? 16 : 32));
    // at most one partial item a request and head, and a row's heads need so many at least
    const int64_t items = kv_heads * std::min(rows * ((group + a.tile_rows - 1) / a.tile_rows), batch + rows * group / a.tile_rows);
    const int64_t tokens = (a.tile_rows - 2) / group + 2;
    // the longest item, in keys
    const int64_t longest = std::min(std::min(window, capacity) + tokens + 63, capacity) + num_globals;
    // Long items are cut wherever a CTA's share of the line ends, and merged by a second kernel;
    // short ones (a band) stay whole, which saves that launch.
    // Many long items of many rows balance by themselves, and their parts are large.
    // Measured (cut | whole, us; contexts of 16K, 32 / 8 heads of 128): one token of 1 request, window 1024, 1400
    // and 2048: 16 | 14, 16 | 17, 16 | 22; of 8 requests 17 | 15, 18 | 18, 19 | 22; of 64 requests 39 | 26, 46 | 43, 54 | 45
    // (from 4096 on 81 | 77).  Chunks, fewer items than 4 an SM, 32K contexts: 8 items of a window of 8192 76 | 209, 256
    // items 461 | 412, of whole contexts 1483 | 1552; 1024 whole contexts 5404 | 5365.  A few chunks with a window
    // little above kWholeKeys would be better whole (32 items, 2048: 148 | 65): their parts cost more than they save.
    a.split = longest > kWholeKeys && (!chunk || items < 4 * kSms);
    // A step of 64 keys shares what it costs besides its keys (waiting, issuing, the vote on the maximum),
    // where the scores of 64 leave the registers for it and items are long enough to fill the warps.
    a.tile_keys = chunk ? kChunkKeys : (a.tile_rows == 8 && a.split ? 64 : 32);
    // Shares of at least 64, 256 and 1024 keys: one token of 4 requests of 2000 keys in 17, 13 and 16 us, of one of
    // 8000 in 16, 15 and 18; of longer ones alike.
    a.min_tiles = 256 / a.tile_keys;
    const int per_sm = chunk ? 1 : ctas_per_sm((int)head_dim, a.tile_rows, a.tile_keys);
    a.items = std::min<int64_t>(items, 0x7fffffff);
    a.ctas = (int)(a.split || chunk ? kSms * per_sm : std::min<int64_t>(items, (int64_t)kSms * per_sm));
    if (a.split) {
        a.part_o = (size_t)a.ctas * 2 * a.tile_rows * head_dim * sizeof(float);
        a.part_ml = (size_t)a.ctas * 2 * a.tile_rows * sizeof(float2);
        a.cuts = items > a.ctas ? (size_t)a.ctas * sizeof(Cut) : 0;
    }
    return a;
}

cudaError_t launch_attention(int d, int tile_rows, int tile_keys, const AttnParams& p, const Globals& g,
                             cudaStream_t stream) {
    return d == 64 ? attention_rows<64>(tile_rows, tile_keys, p, g, stream)
                   : attention_rows<128>(tile_rows, tile_keys, p, g, stream);
}

}  // namespace kv4
}  // namespace lca
