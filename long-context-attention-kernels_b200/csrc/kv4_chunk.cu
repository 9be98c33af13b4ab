// kv4_chunk.cu -- attention of many new tokens a request (a prompt's chunk) over the paged 4-bit KV
// cache, on tcgen05.  Mathematics as in kv4_attention.cu: products over the exact integers c - z,
// scales outside them in fp32.  Q enters as it is, in its own type, which K then shares (the integers
// are exact in bf16 too); V and the weights are fp16.
//
// A CTA takes 256 query rows (tokens x the heads of a group) of one KV head at a time, as two
// tiles A and B of 128 rows, over tiles of 64 keys:
//   unpack warps (4)   a block of 16 keys each: codes from global memory two tiles ahead, as fp16
//                      c - z into a ring of swizzled K and V tiles; scales into a small table
//   MMA warp (1 lane)  S = Q K^T into one of two buffers in TMEM, then O += W V of the tile before, W
//                      read from TMEM where it lies over its S
//   softmax warps (8)  a thread per row: scores times scales, the running maximum, weights to fp16
//   query warps (3)    the next item's query rows into the other of two buffers, and what the softmax
//                      warps need to know of the item (found by themselves it took them 2800 cycles an item,
//                      and registers of their loop)
// Barriers with one phase per tile of one parity (n & 1), so that a wait for tile n - 1 cannot be
// answered by a phase before or after it.
// A tile of codes is unpacked once for 256 rows, and the products of one tile run under
// the softmax of the other.  V is held with the elements of each group of 8 in the order 0 4 1 5 2 6
// 3 7, in which the codes come out of a word most cheaply; the output is put back in order as it
// is read.
#include <algorithm>

#include "kv4_attention.cuh"

namespace lca {
namespace kv4 {
namespace {

constexpr int kHalfRows = 128;            // rows of a tile A or B
constexpr int kKeys = kChunkKeys;         // keys of a tile
// unpacked tiles: with two, a tile could only be unpacked once the product of the one before the last was
// done, and the scores came late (a fifth more time)
constexpr int kRing = 3;
constexpr int kSoftmaxWarps = 8, kUnpackWarps = 4, kMmaWarp = kSoftmaxWarps + kUnpackWarps, kQueryWarps = 3;
constexpr int kThreads = 512;  // four warpgroups: softmax A and B, unpacking, products and queries
// registers a thread of each: 2 * 184 + 80 + 64 = 4 * 128, what the block is launched with
constexpr int kSoftmaxRegs = 184, kUnpackRegs = 80, kMmaRegs = 64;
constexpr uint32_t kTmemCols = 512;

template <int D>
struct Cfg {
    static constexpr int Q_PANEL = kHalfRows * 128, KV_PANEL = kKeys * 128;  // 64 elements of every row
    static constexpr int Q_BYTES = D / 64 * Q_PANEL, KV_BYTES = D / 64 * KV_PANEL;
    static constexpr int OFF_KV = 4 * Q_BYTES;  // two buffers of A and B
    static constexpr int OFF_TABLE = OFF_KV + kRing * 2 * KV_BYTES;  // [kRing][3][kKeys] sk scale log2(e), log2 sv, sv
    static constexpr int OFF_HAVE = OFF_TABLE + kRing * 3 * kKeys * 4;  // [kRing][4] keys that are there, and global ones
    static constexpr int OFF_MOST = OFF_HAVE + kRing * 16;  // [kRing][4] greatest log2 sv of a block
    static constexpr int OFF_LOST = OFF_MOST + kRing * 16;  // [kRing][4] keys whose scale of V is not finite
    static constexpr int OFF_BAR = OFF_LOST + kRing * 16;
    static constexpr int OFF_REST = OFF_BAR + 8 * (17 + 2 * kRing);  // Rest, below
};

// The items of this CTA, in order; the warps that feed the others walk them for themselves, the softmax
// warps get each from the query warps with its queries.
struct Walk {
    Place here;
    Request r;
    long long at, end;
    int head, q_tile, t0, t1;  // q_tile -1: not placed within the request yet
};

struct Item {
    int q0, rows, first_pos;            // the request's first row, rows, and position of the first
    int head, q_tile, t0, tiles, whole; // this one's KV head, rows and tiles [t0, t0 + tiles)
    int first, band;                    // first tile of its band, and tiles of that
    int part;                           // where its part goes: 0 or 1
    int there;                          // 0: no more items
};

// What else is in shared memory: all of it dynamic, as only so three tiles fit next to 256 rows of 128.
struct Rest {
    Item items[2];
    long long scratch[kThreads / 32];
    Place found;
    uint32_t tmem;
    int abort;
};

template <int D>
constexpr int kSmem = Cfg<D>::OFF_REST + (int)sizeof(Rest);
static_assert(Cfg<128>::OFF_REST % alignof(Rest) == 0 && Cfg<64>::OFF_REST % alignof(Rest) == 0, "alignment");
static_assert(kSmem<128> <= 232448, "shared memory of a CTA");

template <int ROWS, int TILE>
__device__ __forceinline__ Place locate_warp(const AttnParams& p, const Globals& g, int from, long long start, long long at) {
    const int lane = threadIdx.x & 31;
    for (int b0 = from; b0 < p.batch; b0 += 32) {
        const Request one = request_of<ROWS, TILE>(p, g, b0 + lane);
        const long long mine = line_of(p, one);
        long long inc = mine;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const long long u = __shfl_up_sync(kAll, inc, o);
            if (lane >= o) inc += u;
        }
        const uint32_t hit = __ballot_sync(kAll, at < start + inc);
        if (hit) {
            const int who = __ffs(hit) - 1;
            Place r = {b0 + who, __shfl_sync(kAll, start + inc - mine, who), {}};
            r.r.q0 = __shfl_sync(kAll, one.q0, who);
            r.r.len = __shfl_sync(kAll, one.len, who);
            r.r.rows = __shfl_sync(kAll, one.rows, who);
            r.r.q_tiles = __shfl_sync(kAll, one.q_tiles, who);
            r.r.tiles = __shfl_sync(kAll, one.tiles, who);
            return r;
        }
        start += __shfl_sync(kAll, inc, 31);
    }
    return {p.batch, start, {0, 0, 0, 0, 1}};
}

// The next item (or part of one) of the walk, or false.
__device__ __forceinline__ bool next_item(const AttnParams& p, const Globals& g, Walk& w) {
    while (w.at < w.end && w.here.b < p.batch) {
        const long long stop = w.here.start + line_of(p, w.r);
        if (w.at >= stop) {
            w.here = locate_warp<kChunkRows, kKeys>(p, g, w.here.b + 1, stop, w.at);
            w.r = w.here.r;
            w.q_tile = -1;
            continue;
        }
        if (w.q_tile >= 0) {  // the item after the last one, which ended where this one begins
            w.t0 = 0;
            if (++w.q_tile == w.r.q_tiles) {
                w.q_tile = 0;
                ++w.head;
            }
        } else {
            const long long in = w.at - w.here.start;
            const int item = in == 0 ? 0 : (int)divide(in, w.r.tiles);
            w.t0 = (int)(in - (long long)item * w.r.tiles);
            if (!p.split && w.t0 > 0) {  // whole items only: this one belongs to the CTA before
                w.at = w.here.start + (long long)(item + 1) * w.r.tiles;
                continue;
            }
            w.head = item == 0 ? 0 : item / w.r.q_tiles;
            w.q_tile = item - w.head * w.r.q_tiles;
        }
        w.t1 = p.split ? (int)min((long long)w.r.tiles, w.t0 + (w.end - w.at)) : w.r.tiles;
        return true;
    }
    return false;
}

// Codes of a word minus the zero point, as pairs in their own order (0 1, 2 3, 4 5, 6 7), in fp16 or bf16:
// 0x6400 | c is 1024 + c in the one, 0x4300 | c is 128 + c in the other.
template <bool BF16>
__device__ __forceinline__ uint4 codes_in_order(uint32_t w, uint32_t zero) {  // zero: 0x10001 times the zero point
    const uint32_t a = __byte_perm(w, w << 12, 0x7610), b = __byte_perm(w, w >> 4, 0x7632);
    const uint32_t magic = BF16 ? 0x43004300u : 0x64006400u, z = magic + zero;
    auto pair = [&](uint32_t v) {
        const uint32_t x = and_or(v, 0x000f000fu, magic);
        uint32_t y;
        if (BF16)
            asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(y) : "r"(x), "r"(z));
        else
            y = hsub2(x, z);
        return y;
    };
    return make_uint4(pair(a), pair(a >> 8), pair(b), pair(b >> 8));
}

__device__ __forceinline__ float max_of_warp(float x) {
    float y;
    asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
    return y;
}

// 16 bytes to shared memory; `valid` false writes zeros and reads nothing.
__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src, bool valid) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0)
                 : "memory");
}

// One row of 64 keys' bits below key index n.
__device__ __forceinline__ uint64_t bits_below(int n) { return n <= 0 ? 0ull : (n >= 64 ? ~0ull : (1ull << n) - 1); }

// Where element e of a group of 8 lies in the order 0 4 1 5 2 6 3 7.
__device__ __forceinline__ constexpr int place(int e) { return e < 4 ? 2 * e : 2 * e - 7; }

// 32 columns of this thread's row of O, times `inv`; zeros where there is nothing to read.
__device__ __forceinline__ void read_out(float (&x)[32], uint32_t taddr, bool some, bool any, float inv) {
    if (any) {  // the same in the whole warp
        ptx::tmem_ld32(taddr, x);
        ptx::tmem_wait_ld();
    }
#pragma unroll
    for (int j = 0; j < 32; ++j) x[j] = some ? x[j] * inv : 0.f;
}

template <int D, bool BF16, bool SPLIT_W>
__global__ void __launch_bounds__(kThreads, 1) kv4_chunk(const AttnParams p, const __grid_constant__ Globals g) {
    using C = Cfg<D>;
    extern __shared__ __align__(1024) uint8_t smem[];
    float* table = reinterpret_cast<float*>(smem + C::OFF_TABLE);
    uint32_t* have_at = reinterpret_cast<uint32_t*>(smem + C::OFF_HAVE);
    uint32_t* lost_at = reinterpret_cast<uint32_t*>(smem + C::OFF_LOST);
    float* most_at = reinterpret_cast<float*>(smem + C::OFF_MOST);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
    uint64_t *q_full = bars, *q_free = bars + 2, *kv_full = bars + 4, *kv_free = kv_full + kRing, *s_full = kv_free + kRing,
             *p_full = s_full + 4, *pv_done = p_full + 4, *drain = pv_done + 4;
    Rest& rest = *reinterpret_cast<Rest*>(smem + C::OFF_REST);
    const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            ptx::mbar_init(&q_full[i], kQueryWarps);
            ptx::mbar_init(&q_free[i], kSoftmaxWarps + 1);  // and the MMA warp
        }
        for (int i = 0; i < kRing; ++i) {
            ptx::mbar_init(&kv_full[i], kUnpackWarps);
            ptx::mbar_init(&kv_free[i], 1);
        }
        for (int i = 0; i < 4; ++i) {
            ptx::mbar_init(&s_full[i], 1);
            ptx::mbar_init(&p_full[i], 4);
            ptx::mbar_init(&pv_done[i], 1);
        }
        ptx::mbar_init(drain, 1);
        rest.abort = 0;
        ptx::fence_mbar_init();
    }
    ptx::griddep_wait();
    Walk walk;
    long long per;
    {
        const Share share = share_of<kChunkRows, kKeys, kThreads>(p, g, rest.scratch, &rest.found);
        if (p.cuts != nullptr && threadIdx.x == 32 * (kMmaWarp + 1)) p.cuts[blockIdx.x].end = 0;  // until it cuts one off
        if (share.at >= share.end) return;
        per = share.per;
        walk.at = share.at;
        walk.end = share.end;
        walk.here = share.here;
        walk.r = share.here.r;
        walk.q_tile = -1;
    }
    const long long line_at = walk.at;
    if (warp == kMmaWarp) {
        ptx::tmem_alloc(&rest.tmem, kTmemCols);
        ptx::tmem_relinquish();
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem = rest.tmem;

    bool ok = true;
    auto wait = [&](uint64_t* bar, int parity) {
        if (ok) ok = ptx::mbar_wait(bar, (uint32_t)parity & 1u, &rest.abort, p.err_word, LCA_DEVERR_TIMEOUT_CACHE, p.wait_ns);
    };
    auto wait_all = [&](uint64_t* bar, int parity) {  // for a whole warp: every lane learns the same
        if (__all_sync(kAll, ok && ptx::mbar_test(bar, (uint32_t)parity & 1u))) return;  // a third of a wait's time
        wait(bar, parity);
        ok = __all_sync(kAll, ok);
    };
    auto tiles_of = [&](Span& s) {  // whole or partial item: its tiles [t0, t0 + n)
        s = span_of<kChunkRows, kKeys>(p, g, walk.r, walk.q_tile);
        return max(0, min(walk.t1, s.band + s.gathered) - walk.t0);
    };
    int n = 0;  // tiles since the start, the same count in every role

    if (warp >= kMmaWarp) {
        ptx::setmaxnreg_dec<kMmaRegs>();
    } else if (warp >= kSoftmaxWarps) {
        ptx::setmaxnreg_dec<kUnpackRegs>();
    } else {
        ptx::setmaxnreg_inc<kSoftmaxRegs>();
    }
    int items = 0;  // items since the start: query buffer items & 1, the same in every role
    if (warp > kMmaWarp) {
        // ============================================================ queries
        // D / 8 lanes a row, 16 bytes each, copied asynchronously into the swizzled tile.  The rows' addresses
        // are found 32 at a time, a lane each (row by row in every lane they took 16000 cycles, which the
        // first item waits for).
        constexpr int LANES = D / 8, AT_ONCE = 32 / LANES;
        const int piece = lane % LANES, sub = lane / LANES;
        while (ok && next_item(p, g, walk)) {
            Span span;
            const int tiles = tiles_of(span);
            if (p.cuts != nullptr && walk.t0 == 0 && walk.t1 < walk.r.tiles && warp == kMmaWarp + 1 && lane == 0)
                p.cuts[blockIdx.x] = {walk.at + walk.r.tiles, per, walk.at != line_at, walk.r.q0, walk.r.rows, walk.head, walk.q_tile};
            const int part = walk.at != line_at;
            walk.at += walk.t1 - walk.t0;
            const int buf = items & 1;
            if (items >= 2) wait_all(&q_free[buf], items / 2 - 1);
            if (!ok) break;
            if (warp == kMmaWarp + 1 && lane == 0)
                rest.items[buf] = {walk.r.q0, walk.r.rows, walk.r.len - p.per_group(walk.r.rows), walk.head, walk.q_tile, walk.t0, tiles,
                                walk.t0 == 0 && walk.t1 == walk.r.tiles, span.first, span.band, part, 1};
            const uint32_t to = ptx::smem_u32(smem + 2 * buf * C::Q_BYTES + (piece >> 3) * C::Q_PANEL);
            const uint16_t* src = static_cast<const uint16_t*>(p.q) + (long long)walk.r.q0 * p.q_token +
                                  (long long)walk.head * p.group * p.q_head;
#pragma unroll 1
            for (int row0 = 0; row0 < kChunkRows && tiles > 0; row0 += 32 * kQueryWarps) {
                // a lane finds one row, number lane of this warp's 32
                const int mine = row0 + 32 * (warp - kMmaWarp - 1) + lane, x = walk.q_tile * kChunkRows + mine;
                const int tok = p.per_group(x);
                const unsigned long long from =
                    x < walk.r.rows ? reinterpret_cast<unsigned long long>(src + tok * p.q_token + (x - tok * p.group) * p.q_head) : 0;
                if (mine - lane >= kChunkRows) break;  // the same in the whole warp
#pragma unroll 8
                for (int k = 0; k < LANES; ++k) {
                    const int which = AT_ONCE * k + sub, row = mine - lane + which, in = row & (kHalfRows - 1);
                    const unsigned long long at = __shfl_sync(kAll, from, which);
                    cp_async_16(to + (row / kHalfRows) * C::Q_BYTES + in * 128 + (((piece & 7) ^ (in & 7)) << 4),
                                at != 0 ? reinterpret_cast<const void*>(at + 16 * piece) : p.q, at != 0);
                }
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
            ptx::fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(&q_full[buf]);
            ++items;
        }
        if (items >= 2) wait_all(&q_free[items & 1], items / 2 - 1);
        if (ok) {
            if (warp == kMmaWarp + 1 && lane == 0) rest.items[items & 1].there = 0;
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(&q_full[items & 1]);
        }
    } else if (warp == kMmaWarp) {
        // ============================================================ products
        const uint32_t hi = ptx::smem_desc_sw128_hi(1024);
        const uint32_t idesc_s = ptx::idesc_f16(BF16, kHalfRows, kKeys, false);
        const uint32_t idesc_o = ptx::idesc_f16(false, kHalfRows, D, true);
        auto accumulate = [&](int m, bool first) {  // O += W V of tile m
            const uint32_t v = ptx::smem_u32(smem + C::OFF_KV + (m % kRing) * 2 * C::KV_BYTES + C::KV_BYTES);
            const uint32_t v_lo = ptx::smem_desc_sw128_lo(v, C::KV_PANEL);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                wait(&p_full[2 * h + (m & 1)], m >> 1);
                if (!ok) return;
                ptx::tc_fence_after();
                const uint32_t o = tmem + 256 * h, w = tmem + 256 * h + 128 + 64 * (m & 1);
#pragma unroll
                for (int part = 0; part < (SPLIT_W ? 2 : 1); ++part)
#pragma unroll
                    for (int k = 0; k < kKeys / 16; ++k)
                        ptx::mma_f16_ts(o, w + 32 * part + 8 * k, ptx::desc_join(v_lo + ((16 * k * 128) >> 4), hi), idesc_o,
                                        !first || part > 0 || k > 0);
                ptx::mma_commit(&pv_done[2 * h + (m & 1)]);
            }
            ptx::mma_commit(&kv_free[m % kRing]);
        };
        while (ok && next_item(p, g, walk)) {
            Span span;
            const int tiles = tiles_of(span);
            walk.at += walk.t1 - walk.t0;
            if (lane == 0) {
                const uint8_t* q_tile = smem + 2 * (items & 1) * C::Q_BYTES;
                wait(&q_full[items & 1], items >> 1);
                if (ok) ptx::mbar_arrive(&q_free[items & 1]);  // seen: no later phase can complete before it was
                for (int i = 0; i < tiles && ok; ++i, ++n) {
                    wait(&kv_full[n % kRing], n / kRing);
                    if (!ok) break;
                    ptx::tc_fence_after();
                    const uint32_t k_lo =
                        ptx::smem_desc_sw128_lo(ptx::smem_u32(smem + C::OFF_KV + (n % kRing) * 2 * C::KV_BYTES), 0);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t q_lo = ptx::smem_desc_sw128_lo(ptx::smem_u32(q_tile + h * C::Q_BYTES), 0);
#pragma unroll
                        for (int k = 0; k < D / 16; ++k)
                            ptx::mma_f16_ss(tmem + 256 * h + 128 + 64 * (n & 1),
                                            ptx::desc_join(q_lo + (((k >> 2) * C::Q_PANEL + (k & 3) * 32) >> 4), hi),
                                            ptx::desc_join(k_lo + (((k >> 2) * C::KV_PANEL + (k & 3) * 32) >> 4), hi), idesc_s,
                                            k > 0);
                        ptx::mma_commit(&s_full[2 * h + (n & 1)]);
                    }
                    if (i > 0) accumulate(n - 1, i == 1);
                }
                if (ok && tiles > 0) accumulate(n - 1, tiles == 1);
            }
            ++items;
            ok = __shfl_sync(kAll, (int)ok, 0) != 0;
        }
        if (lane == 0) {  // whatever was issued has finished before the tiles and TMEM go
            ptx::mma_commit(drain);
            ptx::mbar_wait(drain, 0, nullptr, p.err_word, LCA_DEVERR_TIMEOUT_CACHE, p.wait_ns);
        }
        __syncwarp();
    } else if (warp >= kSoftmaxWarps) {
        // ============================================================ unpacking
        const int w = warp - kSoftmaxWarps, row = lane & 15, side = lane >> 4;
        const float factor = p.scale * kLog2e;
        constexpr int CHUNKS = D / 64;  // 16-byte pieces of a code row per lane
        struct Raw {
            uint4 k[CHUNKS], v[CHUNKS];
            uint32_t word, have;
        };
        while (ok && next_item(p, g, walk)) {
            Span span;
            const int tiles = uniform(tiles_of(span)), t0 = uniform(walk.t0), band = uniform(span.band);
            const int32_t* pages = p.table + (long long)walk.here.b * p.width;
            walk.at += walk.t1 - walk.t0;
            // the pool's block of a position, or -1
            auto block_at = [&](int block) {
                const int page_at = p.pool.per_page(block), page = pages[page_at];
                if ((unsigned)page >= (unsigned)p.pool.pages) return -1;
                return (page * p.pool.kv_heads + walk.head) * p.pool.page_blocks + block - page_at * p.pool.page_blocks;
            };
            int where = -1;  // blocks of this warp in 32 tiles, a lane per tile
            auto load = [&](int i, Raw& x) {
                if (i >= tiles) return;
                if ((i & 31) == 0) {
                    const int block = 4 * (span.first + t0 + i + lane) + w;
                    where = i + lane < tiles && t0 + i + lane < band && block <= span.hi / kBlock ? block_at(block) : -1;
                }
                int at, of = row;
                if (t0 + i < band) {
                    at = __shfl_sync(kAll, where, i & 31);
                } else {
                    const int k = (t0 + i - band) * kKeys + kBlock * w + row;
                    at = -1;
                    if (k < span.globals) {
                        at = block_at(g.at[k] / kBlock);
                        of = g.at[k] % kBlock;
                    }
                }
                // the block's keys that are there, and above them those that are global and in the band
                uint32_t glob = 0;
                if (p.num_globals > 0 && t0 + i < band) {
                    const int key = (span.first + t0 + i) * kKeys + kBlock * w + row, k = lower_bound(g.at, p.num_globals, key);
                    glob = __ballot_sync(kAll, k < p.num_globals && g.at[k] == key);
                }
                x.have = (__ballot_sync(kAll, at >= 0) & 0xffffu) | (glob << 16);
                const uint8_t* src = p.pool.data + (long long)at * block_bytes(D);
                if (at >= 0) {
                    x.word = *reinterpret_cast<const uint32_t*>(src + (side ? v_words_at(D) : k_words_at(D)) + 4 * of);
#pragma unroll
                    for (int c = 0; c < CHUNKS; ++c) {
                        x.k[c] = *reinterpret_cast<const uint4*>(src + of * row_bytes(D) + 16 * (side + 2 * c));
                        x.v[c] = *reinterpret_cast<const uint4*>(src + v_codes_at(D) + of * row_bytes(D) + 16 * (side + 2 * c));
                    }
                } else {
                    x.word = 0;
#pragma unroll
                    for (int c = 0; c < CHUNKS; ++c) x.k[c] = x.v[c] = make_uint4(0, 0, 0, 0);
                }
            };
            auto store = [&](int i, const Raw& x) {
                if (i >= tiles) return;
                const int slot = n % kRing;
                if (n >= kRing) wait_all(&kv_free[slot], n / kRing - 1);
                if (!ok) return;
                float* sk = table + slot * 3 * kKeys;
                const float scale = __uint_as_float(x.word & ~15u);
                float lam = 0.f;
                if (side == 0) {
                    sk[kBlock * w + row] = scale * factor;
                } else {
                    lam = fmaxf(lg2(fabsf(scale)), kLeast);
                    sk[kKeys + kBlock * w + row] = lam;
                    sk[2 * kKeys + kBlock * w + row] = fabsf(scale) < INFINITY ? scale : 0.f;
                }
                // a weight of 0 times such a scale would not be 0, so it is kept out of the products
                const uint32_t lost = __ballot_sync(kAll, side == 1 && ((x.have >> row) & 1) && !(fabsf(scale) < INFINITY)) >> 16;
                const bool counts = side == 1 && ((x.have >> row) & 1);
                const float most = lost ? INFINITY : max_of_warp(counts ? lam : -INFINITY);
                if (lane == 0) {
                    most_at[slot * 4 + w] = most;
                    lost_at[slot * 4 + w] = lost;
                    have_at[slot * 4 + w] = x.have;
                }
                const uint32_t word_k = __shfl_sync(kAll, x.word, row), word_v = __shfl_sync(kAll, x.word, row + 16);
                const Zero zv = zero_pair((word_v & 15u) * 0x10001u);
                uint8_t* k_tile = smem + C::OFF_KV + slot * 2 * C::KV_BYTES;
                const int r = kBlock * w + row;
#pragma unroll
                for (int c = 0; c < CHUNKS; ++c) {
                    const uint32_t kw[4] = {x.k[c].x, x.k[c].y, x.k[c].z, x.k[c].w};
                    const uint32_t vw[4] = {x.v[c].x, x.v[c].y, x.v[c].z, x.v[c].w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        // word 4 (side + 2c) + j of the row: 8 elements, 16 bytes of a panel's row
                        const int word = 4 * (side + 2 * c) + j;
                        uint8_t* to = k_tile + (word >> 3) * C::KV_PANEL + r * 128 + (((word & 7) ^ (r & 7)) << 4);
                        *reinterpret_cast<uint4*>(to) = codes_in_order<BF16>(kw[j], (word_k & 15u) * 0x10001u);
                        *reinterpret_cast<uint4*>(to + C::KV_BYTES) =
                            make_uint4(codes_pair(vw[j], 0, zv), codes_pair(vw[j], 1, zv), codes_pair(vw[j], 2, zv),
                                       codes_pair(vw[j], 3, zv));
                    }
                }
                ptx::fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(&kv_full[slot]);
                ++n;
            };
            Raw a, b;
            load(0, a);
            load(1, b);
#pragma unroll 1
            for (int i = 0; i < tiles && ok; ++i) {  // (two copies of this in one turn cost more in fetching code)
                store(i, a);
                a = b;
                load(i + 2, b);
            }
        }
    } else {
        // ============================================================ softmax
        const int h = warp >> 2, in_half = 32 * (warp & 3) + lane;
        const uint32_t mine = tmem + 256 * h + ((uint32_t)(32 * (warp & 3)) << 16);
        while (true) {
            wait_all(&q_full[items & 1], items >> 1);
            if (!ok) break;
            const Item& it = rest.items[items & 1];  // and its queries' buffer: this warp's until it arrives at q_free
            if (!it.there) break;
            const int tiles = uniform(it.tiles), t0 = uniform(it.t0), first = uniform(it.first), band = uniform(it.band);
            const int of = it.q_tile * kChunkRows + h * kHalfRows + in_half;
            const bool valid = of < it.rows;
            const int pos = valid ? it.first_pos + p.per_group(of) : -1;
            int row_lo = max(0, pos - p.window);
            float top = -INFINITY;
            bool finite = true, any = false, lost = false;  // the row of q; whether it sees a key, and one of V lost
            int from_key = 0, to_key = 0;  // tiles that begin here are visible to all rows of the warp
            uint64_t sum2 = ptx::f2_pack(0.f, 0.f);
            if (tiles > 0) {
                if (p.num_globals > 0 && first == 0 && valid) {
                    const int k = lower_bound(g.at, p.num_globals, pos);
                    if (k < p.num_globals && g.at[k] == pos) row_lo = 0;
                }
                from_key = __reduce_max_sync(kAll, valid ? row_lo : 0);
                to_key = __reduce_min_sync(kAll, valid ? pos : 0x7fffffff) - kKeys + 1;
                const uint8_t* q_row = smem + (2 * (items & 1) + h) * C::Q_BYTES + in_half * 128;
                uint32_t most = 0;
#pragma unroll
                for (int i = 0; i < D / 8; ++i) {  // in any order of the row's pieces
                    const uint4 v = *reinterpret_cast<const uint4*>(q_row + (i >> 3) * C::Q_PANEL + (((i ^ in_half) & 7) << 4));
                    most = __vmaxu2(most, __vmaxu2(__vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu),
                                                   __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu)));
                }
                finite = max(most & 0xffffu, most >> 16) < (BF16 ? 0x7f80u : 0x7c00u);
            }

#pragma unroll 1
            for (int i = 0; i < tiles; ++i, ++n) {
                const int slot = n % kRing, buf = n & 1, tile = t0 + i;
                // the tile's table is complete since its scores are; its barrier makes it visible here
                const bool scores = ptx::mbar_test(&s_full[2 * h + buf], (uint32_t)(n >> 1) & 1u);
                const bool tables = ptx::mbar_test(&kv_full[slot], (uint32_t)(n / kRing) & 1u);
                if (!__all_sync(kAll, ok && scores && tables)) {
                    wait_all(&s_full[2 * h + buf], n >> 1);
                    wait_all(&kv_full[slot], n / kRing);
                    if (!ok) break;
                }
                ptx::tc_fence_after();
                uint64_t s[kKeys / 2];  // pairs of keys
                const uint32_t s_at = mine + 128 + 64 * buf;
                float x0[32], x1[32];
                ptx::tmem_ld32(s_at, x0);
                ptx::tmem_ld32(s_at + 32, x1);
                // what says which keys count comes while the scores do
                const uint4 hs = *reinterpret_cast<const uint4*>(have_at + slot * 4);
                ptx::tmem_wait_ld();
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    s[j] = ptx::f2_pack(x0[2 * j], x0[2 * j + 1]);
                    s[16 + j] = ptx::f2_pack(x1[2 * j], x1[2 * j + 1]);
                }
                const ulonglong2* sk = reinterpret_cast<const ulonglong2*>(table + slot * 3 * kKeys);
                const ulonglong2 *lam = sk + kKeys / 4, *sv = lam + kKeys / 4;
#pragma unroll
                for (int j = 0; j < kKeys / 4; ++j) {
                    const ulonglong2 a = sk[j];
                    s[2 * j] = ptx::f2_mul(s[2 * j], a.x);
                    s[2 * j + 1] = ptx::f2_mul(s[2 * j + 1], a.y);
                }

                // ---- visibility
                const bool in_band = tile < band;
                const int key0 = (first + tile) * kKeys;
                const uint64_t have = (uint64_t)__byte_perm(hs.x, hs.y, 0x5410) | ((uint64_t)__byte_perm(hs.z, hs.w, 0x5410) << 32);
                const bool full = have == ~0ull && (!in_band || (key0 >= from_key && key0 <= to_key));
                uint64_t seen = ~0ull;
                if (full) {
                    any = true;
                } else {
                    const uint64_t glob = (uint64_t)__byte_perm(hs.x, hs.y, 0x7632) | ((uint64_t)__byte_perm(hs.z, hs.w, 0x7632) << 32);
                    if (in_band)
                        seen = bits_below(pos - key0 + 1) & (~bits_below(row_lo - key0) | glob);
                    else
                        seen = pos >= 0 ? ~0ull : 0ull;
                    seen &= have;
                    any |= seen != 0;
#pragma unroll
                    for (int j = 0; j < kKeys / 2; ++j) {
                        const float x = (seen >> (2 * j)) & 1 ? ptx::f2_lo(s[j]) : -INFINITY;
                        const float y = (seen >> (2 * j + 1)) & 1 ? ptx::f2_hi(s[j]) : -INFINITY;
                        s[j] = ptx::f2_pack(x, y);
                    }
                }

                // ---- running maximum of x + log2(sv): the sum of the two maxima is no less, at a third of the
                // instructions, and says whether any row may have to move.  Whether and where to is then
                // found from the keys that the row sees, and from nothing else.
                float peak = INFINITY, peak1 = -INFINITY;
                if (i > 0) {  // the first tile always moves it
                    const float4 most4 = *reinterpret_cast<const float4*>(most_at + slot * 4);
                    peak = -INFINITY;
#pragma unroll
                    for (int j = 0; j < kKeys / 4; ++j) {
                        peak = ptx::fmax3(peak, ptx::f2_lo(s[2 * j]), ptx::f2_hi(s[2 * j]));
                        peak1 = ptx::fmax3(peak1, ptx::f2_lo(s[2 * j + 1]), ptx::f2_hi(s[2 * j + 1]));
                    }
                    peak = fmaxf(peak, peak1) + fmaxf(ptx::fmax3(most4.x, most4.y, most4.z), most4.w);
                }
                if (__any_sync(kAll, peak > top + kRise)) {
                    const uint4 ls = *reinterpret_cast<const uint4*>(lost_at + slot * 4);
                    lost |= (seen & ((uint64_t)(ls.x | ls.y << 16) | ((uint64_t)(ls.z | ls.w << 16) << 32))) != 0;
                    peak = peak1 = -INFINITY;
#pragma unroll
                    for (int j = 0; j < kKeys / 4; ++j) {
                        const ulonglong2 a = lam[j];
                        const uint64_t u = ptx::f2_add(s[2 * j], a.x), v = ptx::f2_add(s[2 * j + 1], a.y);
                        peak = ptx::fmax3(peak, ptx::f2_lo(u), ptx::f2_hi(u));
                        peak1 = ptx::fmax3(peak1, ptx::f2_lo(v), ptx::f2_hi(v));
                    }
                    peak = fmaxf(peak, peak1);
                    const bool rise = peak > top + kRise;
                    const float to = rise ? peak - kHead : top;
                    const float half = rise ? ex2_half(top - to) : 1.f, f = half * half;
                    const uint64_t half2 = ptx::f2_pack(half, half);
                    top = to;
                    sum2 = ptx::f2_mul(ptx::f2_mul(sum2, half2), half2);
                    if (__any_sync(kAll, rise) && i > 0) {
                        wait_all(&pv_done[2 * h + ((n - 1) & 1)], (n - 1) >> 1);
                        if (!ok) break;
                        ptx::tc_fence_after();
#pragma unroll 1
                        for (int c = 0; c < D; c += 32) {
                            float x[32];
                            ptx::tmem_ld32(mine + c, x);
                            ptx::tmem_wait_ld();
#pragma unroll
                            for (int j = 0; j < 32; ++j) x[j] *= f;
                            ptx::tmem_st32(mine + c, x);
                        }
                        ptx::tmem_wait_st();
                    }
                }

                // ---- weights
                const float ref = top == -INFINITY ? 0.f : -top;
                const uint64_t ref2 = ptx::f2_pack(ref, ref);
                uint64_t tile2 = ptx::f2_pack(0.f, 0.f);  // the tile's own sum first: a chain of 32 + tiles, not of 32 tiles
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint32_t hi[kKeys / 4], lo[kKeys / 4];
#pragma unroll
                    for (int k = 0; k < kKeys / 4; ++k) {
                        const int j = half * (kKeys / 4) + k;
                        const uint64_t x = ptx::f2_add(s[j], ref2);
                        const uint64_t e = ptx::f2_pack(ptx::ex2(ptx::f2_lo(x)), ptx::ex2(ptx::f2_hi(x)));
                        tile2 = ptx::f2_add(tile2, e);
                        const ulonglong2 v4 = sv[j >> 1];
                        const uint64_t w = ptx::f2_mul(e, (j & 1) ? v4.y : v4.x);
                        const float w0 = ptx::f2_lo(w), w1 = ptx::f2_hi(w);
                        hi[k] = ptx::pack_f16x2(w0, w1);
                        if (SPLIT_W) {
                            const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&hi[k]));
                            lo[k] = ptx::pack_f16x2(w0 - back.x, w1 - back.y);
                        }
                    }
                    ptx::tmem_st16u(s_at + kKeys / 4 * half, hi);
                    if constexpr (SPLIT_W) ptx::tmem_st16u(s_at + kKeys / 2 + kKeys / 4 * half, lo);
                }
                sum2 = ptx::f2_add(sum2, tile2);
                ptx::tmem_wait_st();
                ptx::tc_fence_before();
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(&p_full[2 * h + buf]);
            }

            // ---- the row's output, or its part
            if (ok && tiles > 0) {
                wait_all(&pv_done[2 * h + ((n - 1) & 1)], (n - 1) >> 1);
                ptx::tc_fence_after();
            }
            if (!ok) break;
            float sum = ptx::f2_lo(sum2) + ptx::f2_hi(sum2);
            if (any && !finite) sum = NAN;
            const bool whole = it.whole;
            const int token = p.per_group(of), head = it.head * p.group + of - token * p.group, q0 = it.q0;
            const float inv = lost ? NAN : (whole ? (sum == 0.f ? 0.f : 1.f / sum) : 1.f);
            const long long part = (long long)(2 * blockIdx.x + it.part) * kChunkRows + h * kHalfRows + in_half;
            const long long out_at = ((long long)(q0 + token) * p.heads + head) * D;
            if (valid) {
                if (!whole) {
                    p.part_ml[part] = make_float2(top, sum);
                } else if (p.lse != nullptr) {
                    p.lse[(long long)head * p.rows + q0 + token] = lse_of(top, sum);
                }
            }
            if (whole && p.out_dtype != LCA_DTYPE_F32) {
                // 16-bit rows go through the warp's own rows of the query tile, which nothing reads any more,
                // and leave as whole rows, D / 8 lanes each
                auto stage = [&](int row, int piece) {
                    return reinterpret_cast<uint4*>(smem + (2 * (items & 1) + h) * C::Q_BYTES + (piece >> 3) * C::Q_PANEL +
                                                    (32 * (warp & 3) + row) * 128 + (((piece & 7) ^ (row & 7)) << 4));
                };
#pragma unroll 1
                for (int c = 0; c < D; c += 32) {
                    float x[32];
                    read_out(x, mine + c, tiles > 0 && sum != 0.f, tiles > 0, inv);
#pragma unroll
                    for (int j = 0; j < 32; j += 8) {
                        uint32_t v[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k)  // back from the order 0 4 1 5 2 6 3 7
                            v[k] = p.out_dtype == LCA_DTYPE_F16
                                       ? ptx::pack_f16x2(x[j + place(2 * k)], x[j + place(2 * k + 1)])
                                                                : ptx::pack_bf16x2(x[j + place(2 * k)], x[j + place(2 * k + 1)]);
                        *stage(lane, (c + j) / 8) = make_uint4(v[0], v[1], v[2], v[3]);
                    }
                }
                __syncwarp();
                constexpr int LANES = D / 8, AT_ONCE = 32 / LANES;
#pragma unroll 4
                for (int i = 0; i < LANES; ++i) {
                    const int row = AT_ONCE * i + lane / LANES, piece = lane % LANES;
                    const int to = __shfl_sync(kAll, valid ? (q0 + token) * p.heads + head : -1, row);
                    if (to >= 0)
                        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + (long long)to * D + 8 * piece) = *stage(row, piece);
                }
                __syncwarp();
            } else {
                float* to = whole ? static_cast<float*>(p.out) + out_at : p.part_o + part * D;
#pragma unroll 1
                for (int c = 0; c < D; c += 32) {
                    float x[32];
                    read_out(x, mine + c, tiles > 0 && !(whole && sum == 0.f), tiles > 0, inv);
#pragma unroll
                    for (int j = 0; j < 32; j += 4) {
                        const float* v = x + (j & ~7);
                        const int k = j & 4;
                        if (valid)
                            *reinterpret_cast<float4*>(to + c + j) =
                                make_float4(v[place(k)], v[place(k + 1)], v[place(k + 2)], v[place(k + 3)]);
                    }
                    __syncwarp();
                }
            }
            ptx::tc_fence_before();  // the next item's products overwrite what was read here
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(&q_free[items & 1]);
            ++items;
        }
    }
    ptx::tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc(tmem, kTmemCols);
    }
}

template <int D, bool BF16, bool SPLIT_W>
cudaError_t chunk_of(const AttnParams& p, const Globals& g, cudaStream_t stream) {
    static std::atomic<unsigned long long> done{0};
    cudaError_t e = allow_smem(kv4_chunk<D, BF16, SPLIT_W>, kSmem<D>, done);
    if (e != cudaSuccess) return e;
    return launch_early(kv4_chunk<D, BF16, SPLIT_W>, dim3(p.ctas), kThreads, kSmem<D>, stream, p, g);
}

template <int D>
cudaError_t chunk_types(const AttnParams& p, const Globals& g, cudaStream_t stream) {
    const bool split_w = p.out_dtype != LCA_DTYPE_BF16;
    if (p.bf16) return split_w ? chunk_of<D, true, true>(p, g, stream) : chunk_of<D, true, false>(p, g, stream);
    return split_w ? chunk_of<D, false, true>(p, g, stream) : chunk_of<D, false, false>(p, g, stream);
}

}  // namespace

cudaError_t launch_chunk(int d, const AttnParams& p, const Globals& g, cudaStream_t stream) {
    return d == 64 ? chunk_types<64>(p, g, stream) : chunk_types<128>(p, g, stream);
}

}  // namespace kv4
}  // namespace lca
