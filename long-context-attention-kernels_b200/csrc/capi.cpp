// capi.cpp -- the C ABI (include/lca.h): argument validation with the reference's
// semantics, workspace layout, TMA tensor-map construction and the launch sequence
// gather -> main -> combine on the caller's stream.
#include "lca.h"

#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstddef>
#include <climits>
#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <mutex>
#include <string>
#include <vector>

#include "kv4.h"
#include "swa_kernels.h"
#include "swa_backward.h"

namespace {

thread_local std::string g_last_error;
thread_local cudaEvent_t g_ev_before_main = nullptr;
thread_local cudaEvent_t g_ev_after_main = nullptr;

int fail(int status, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    g_last_error = buf;
    return status;
}

}  // namespace

int lca::report_error(int status, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    g_last_error = buf;
    return status;
}

namespace {

int fail_cuda(cudaError_t e, const char* what) {
    return fail(LCA_ERR_CUDA, "%s: %s (%s)", what, cudaGetErrorName(e), cudaGetErrorString(e));
}

// ------------------------------------------------------------------ device checks

constexpr int kMaxDevices = 64;
std::mutex g_dev_mu;
int g_dev_state[kMaxDevices];          // 0 unknown, 1 ok, -1 unsupported
int* g_dev_err_word[kMaxDevices];      // device address of the error word
int g_dev_sms[kMaxDevices];            // multiprocessor count

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn get_encode_fn() {
    static EncodeTiledFn fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeTiledFn>(p);
    });
    return fn;
}

int check_device(int* dev_out, int** err_word) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return fail_cuda(e, "cudaGetDevice");
    if (dev < 0 || dev >= kMaxDevices) return fail(LCA_ERR_UNSUPPORTED, "device ordinal %d out of range", dev);
    std::lock_guard<std::mutex> lk(g_dev_mu);
    if (g_dev_state[dev] == 0) {
        int major = 0, minor = 0;
        cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev);
        cudaDeviceGetAttribute(&minor, cudaDevAttrComputeCapabilityMinor, dev);
        if (major != 10 || minor != 0) {
            g_dev_state[dev] = -1;
        } else {
            int* addr = nullptr;
            e = lca::error_word_address(&addr);
            if (e != cudaSuccess) return fail_cuda(e, "cudaGetSymbolAddress(error word)");
            g_dev_err_word[dev] = addr;
            cudaDeviceGetAttribute(&g_dev_sms[dev], cudaDevAttrMultiProcessorCount, dev);
            if (g_dev_sms[dev] <= 0) g_dev_sms[dev] = 148;
            g_dev_state[dev] = 1;
        }
    }
    if (g_dev_state[dev] < 0)
        return fail(LCA_ERR_UNSUPPORTED, "device %d is not an sm_100 (B200-class) GPU; this library is built for sm_100a",
                    dev);
    *dev_out = dev;
    *err_word = g_dev_err_word[dev];
    return LCA_OK;
}

// ------------------------------------------------------------------ problem description

// One forward problem: the whole sequence (q_off = 0, n = n_total), or one contiguous
// shard of it.
struct Problem {
    int64_t bh = 0;
    int64_t heads = 1;     // heads per batch (bh = batch * heads)
    bool tok_major = false;  // q, k, v, out are [batch][n][heads][d] (else [batch][heads][n][d])
    int64_t n_total = 0;   // sequence length
    int64_t n = 0;         // local rows of Q / K / V / O
    int64_t q_off = 0;     // absolute index of local row 0
    int64_t d = 0;
    int64_t window = 0;    // clamped to n_total
    int64_t G = 0;         // unique global tokens
    int64_t world = 1;     // shards
    bool sharded = false;
    int dtype = LCA_DTYPE_BF16;
    int out_dtype = LCA_DTYPE_F32;  // type of out (16-bit only through lca_swa_forward_ex)
    bool causal = false;            // LCA_FLAG_CAUSAL (whole-sequence problems only)
    std::vector<int> head_window;   // a radius per head (whole-sequence problems), else empty
    int seg_mode = lca::kSegNone;   // band clipped to segments (lca::MainParams::seg_mode)
    int64_t seg_len = 0;            // kSegEqual: tokens per segment
    std::vector<int> seg_start;     // kSegVarlen: segment starts, then the total
    float scale = 1.f;
    std::vector<int32_t> gl;  // sorted unique global indices (absolute)
    int64_t halo() const { return sharded && world > 1 ? window : 0; }
    // element strides of q / k / v / out: batch, head, row
    int64_t s_b() const { return tok_major ? n * heads * d : heads * n * d; }
    int64_t s_h() const { return tok_major ? d : n * d; }
    int64_t s_n() const { return tok_major ? heads * d : d; }
    int64_t lead() const {
        return sharded ? (window + lca::kTileRows - 1) / lca::kTileRows * lca::kTileRows : window;
    }
};

int check_dtype_dim(int dtype, int64_t head_dim) {
    if (dtype != LCA_DTYPE_F16 && dtype != LCA_DTYPE_BF16)
        return fail(LCA_ERR_UNSUPPORTED, "dtype %d is not supported (fp16 or bf16 inputs)", dtype);
    if (head_dim != 64 && head_dim != 128)
        return fail(LCA_ERR_UNSUPPORTED, "head_dim %lld is not supported (64 or 128)", (long long)head_dim);
    return LCA_OK;
}

// Shape checks shared by every entry point (csrc/bindings.cpp:25-42 restated for a C
// caller), then the global-token list, normalised as the reference's mask builds it.
int parse_common(Problem& P, int dtype, int64_t batch, int64_t heads, int64_t seq_len, int64_t head_dim,
                 int64_t window_size, float scale, const int64_t* global_tokens, int64_t num_global_tokens) {
    int st = check_dtype_dim(dtype, head_dim);
    if (st != LCA_OK) return st;
    if (batch < 0 || heads < 0 || seq_len < 0) return fail(LCA_ERR_INVALID_ARGUMENT, "negative shape");
    if (window_size < 0)
        return fail(LCA_ERR_INVALID_ARGUMENT, "window_size must be >= 0 (got %lld)", (long long)window_size);
    if (seq_len > ((int64_t)1 << 29))
        return fail(LCA_ERR_UNSUPPORTED, "seq_len %lld too large (max 2^29)", (long long)seq_len);
    const int64_t bh = batch * heads;
    if (bh > INT_MAX / 64) return fail(LCA_ERR_UNSUPPORTED, "batch*heads %lld too large", (long long)bh);
    if (num_global_tokens < 0) return fail(LCA_ERR_INVALID_ARGUMENT, "negative global token count");
    if (num_global_tokens > 0 && global_tokens == nullptr)
        return fail(LCA_ERR_INVALID_ARGUMENT, "global_tokens is NULL");
    // Global tokens are validated even for empty problems, as the reference's mask
    // construction would raise on them.
    P.gl.assign((size_t)num_global_tokens + 1, 0);
    int64_t G = 0;
    st = lca_normalize_global_tokens(global_tokens, num_global_tokens, seq_len, P.gl.data(), &G);
    if (st != LCA_OK) return st;
    P.gl.resize((size_t)G);
    P.bh = bh;
    P.heads = heads > 0 ? heads : 1;
    P.n_total = seq_len;
    P.n = seq_len;
    P.q_off = 0;
    P.d = head_dim;
    P.window = std::min(window_size, seq_len);
    P.G = G;
    P.dtype = dtype;
    P.scale = scale;
    return LCA_OK;
}

int parse_shard(Problem& P, const lca_shard_desc* sd, const int64_t* global_tokens, int64_t num_global_tokens) {
    if (sd == nullptr) return fail(LCA_ERR_INVALID_ARGUMENT, "shard descriptor is NULL");
    int st = parse_common(P, sd->dtype, sd->batch, sd->heads, sd->seq_len, sd->head_dim, sd->window_size, sd->scale,
                          global_tokens, num_global_tokens);
    if (st != LCA_OK) return st;
    if (sd->world_size < 1) return fail(LCA_ERR_INVALID_ARGUMENT, "world_size must be >= 1");
    if (sd->rank < 0 || sd->rank >= sd->world_size)
        return fail(LCA_ERR_INVALID_ARGUMENT, "rank %lld outside [0, %lld)", (long long)sd->rank,
                    (long long)sd->world_size);
    if (sd->shard_offset < 0 || sd->shard_len < 1 || sd->shard_offset + sd->shard_len > sd->seq_len)
        return fail(LCA_ERR_INVALID_ARGUMENT, "shard [%lld, %lld) is not inside the sequence of %lld tokens",
                    (long long)sd->shard_offset, (long long)(sd->shard_offset + sd->shard_len), (long long)sd->seq_len);
    const bool last = sd->shard_offset + sd->shard_len == sd->seq_len;
    if (!last && sd->shard_len % lca::kTileRows != 0)
        return fail(LCA_ERR_UNSUPPORTED, "a shard other than the last must hold a multiple of %d tokens (got %lld)",
                    lca::kTileRows, (long long)sd->shard_len);
    if (sd->world_size > 1 && P.window > sd->shard_len)
        return fail(LCA_ERR_UNSUPPORTED,
                    "window %lld exceeds the shard length %lld: halos come from the adjacent shards only",
                    (long long)P.window, (long long)sd->shard_len);
    P.sharded = true;
    P.world = sd->world_size;
    P.n = sd->shard_len;
    P.q_off = sd->shard_offset;
    return LCA_OK;
}

// ------------------------------------------------------------------ workspace layout

constexpr int kMinGrowUnits = 148;  // at least one global-row unit per SM when possible
constexpr size_t kAlign = 1024;

size_t align_up(size_t x, size_t a) { return (x + a - 1) / a * a; }

struct Layout {
    int g_tiles = 0, key_tiles = 0, n_splits = 0, split_tiles = 0;
    size_t grow_bytes = 0;  // one compact global row: [3][bh][d]
    size_t off_sig = 0;     // sequence shards: peer-exchange counters (lca::PeerSignals)
    size_t off_gidx = 0, off_globals = 0, off_po = 0, off_plse = 0;
    size_t off_send = 0, off_recv = 0, halo_block = 0;  // halo_block: one side, [2][bh][halo][d]
    size_t off_rowpart = 0, rowpart_bytes = 0, off_rowpart_all = 0;  // rowpart_all: two buffers
    size_t total = 0;  // bytes the forward needs
    // Optional suffix.  For bf16 inputs: an fp16 copy of V [bh][n][d], of the compact global
    // V rows [G][bh][d] and, for a sequence shard, of the received halo blocks (laid out like
    // the receive region, V planes filled), and a word that says whether some value did not
    // convert without loss that matters (lca_convert_v16).  When none failed, P*V runs once
    // per tile in fp16 instead of twice (bf16 P split into hi + lo).  For every dtype: the
    // word from which the main kernel's CTAs take work units (dynamic scheduling; without
    // it units go round-robin).  The suffix follows every other region (for a shard: after
    // this rank's own regions, so the exchanged regions keep their offsets).
    // total_fast >= total; a workspace of total_fast bytes enables it.
    size_t off_v16 = 0, off_vg16 = 0, off_vh16 = 0, off_v16bad = 0;
    bool has_v16 = false;    // bf16: the suffix holds the fp16 copy of V
    size_t off_counter = 0;  // suffix: the main kernel's work-unit counter (zeroed per launch)
    size_t total_fast = 0;
};

// Split of the keys of the global-row units (all n keys, or the shard's own).  A unit
// covers `split_tiles` key tiles (its two query-tile warpgroups take alternate tiles),
// sized at about twice a band unit's work so units stay similar in length, but shrunk
// until there are enough units to occupy every SM.  Each split yields two partial
// results (even / odd tiles).
//
// For a sequence shard the regions other ranks write come first -- signal counters,
// compact global rows, halo receive blocks, gathered row partials -- and their sizes
// depend only on quantities every rank shares (heads, G, d, window, world), so they sit
// at the same offsets on every rank.  The rank's own regions follow.
Layout make_layout(const Problem& P) {
    Layout L;
    const int64_t bh = P.bh, G = P.G, d = P.d;
    const bool glob = G > 0 && bh > 0 && P.n > 0;
    if (glob) {
        L.g_tiles = (int)((G + lca::kTileRows - 1) / lca::kTileRows);
        L.key_tiles = (int)((P.n + lca::kTileRows - 1) / lca::kTileRows);
        const int64_t band_tiles = (P.lead() + P.window + 2 * lca::kTileRows - 1) / lca::kTileRows + L.g_tiles;
        int64_t split = std::max<int64_t>(4, std::min<int64_t>(64, 4 * band_tiles));
        const int64_t units_per_split_count = bh * L.g_tiles;
        while (split > 2 && units_per_split_count * ((L.key_tiles + split - 1) / split) < kMinGrowUnits) split -= 2;
        split += split & 1;
        L.split_tiles = (int)split;
        L.n_splits = (L.key_tiles + L.split_tiles - 1) / L.split_tiles;
        L.grow_bytes = (size_t)3 * bh * d * 2;
        if (P.sharded) {
            // O [bh][G][d], then LSE [bh][G] padded to 16 bytes (each rank's block in the
            // gathered region stays 16-byte aligned for the merge's float4 loads)
            L.rowpart_bytes = (size_t)bh * G * d * 4 + align_up((size_t)bh * G * 4, 16);
        }
    }
    if (P.halo() > 0 && bh > 0) L.halo_block = (size_t)2 * bh * P.halo() * d * 2;
    const int64_t parts = 2 * (int64_t)L.n_splits;
    size_t off = 0;
    if (P.sharded) {
        L.off_sig = off;
        off = align_up(off + sizeof(lca::PeerSignals), kAlign);
        L.off_globals = off;  // compact rows [G][3 (q, k, v)][bh][d]
        off = align_up(off + (size_t)G * L.grow_bytes, kAlign);
        L.off_recv = off;
        off = align_up(off + 2 * L.halo_block, kAlign);
        L.off_rowpart_all = off;
        off = align_up(off + 2 * L.rowpart_bytes * (size_t)P.world, kAlign);
        // this rank's own regions
        L.off_gidx = off;
        off = align_up(off + sizeof(int) * G, kAlign);
        L.off_po = off;
        off = align_up(off + (size_t)parts * bh * G * d * 4, kAlign);
        L.off_plse = off;
        off = align_up(off + (size_t)parts * bh * G * 4, kAlign);
        L.off_rowpart = off;
        off = align_up(off + L.rowpart_bytes, kAlign);
        L.off_send = off;
        off = align_up(off + 2 * L.halo_block, kAlign);
    } else if (glob) {
        L.off_gidx = off;
        off = align_up(off + sizeof(int) * G, kAlign);
        L.off_globals = off;
        off = align_up(off + (size_t)G * L.grow_bytes, kAlign);
        L.off_po = off;
        off = align_up(off + (size_t)parts * bh * G * d * 4, kAlign);
        L.off_plse = off;
        off = align_up(off + (size_t)parts * bh * G * 4, kAlign);
    }
    L.total = off;
    L.total_fast = off;
    if (P.dtype == LCA_DTYPE_BF16 && bh > 0 && P.n > 0) {
        L.off_v16 = off;
        off = align_up(off + (size_t)bh * P.n * d * 2, kAlign);
        if (glob) {
            L.off_vg16 = off;
            off = align_up(off + (size_t)G * bh * d * 2, kAlign);
        }
        if (L.halo_block > 0) {
            L.off_vh16 = off;
            off = align_up(off + 2 * L.halo_block, kAlign);
        }
        // the word and the work-unit counter sit side by side, so one memset clears both
        L.off_v16bad = off;
        L.off_counter = off + sizeof(int);
        off = align_up(off + 2 * sizeof(int), kAlign);
        L.has_v16 = true;
    } else if (bh > 0 && P.n > 0) {
        L.off_counter = off;
        off = align_up(off + sizeof(unsigned int), kAlign);
    }
    L.total_fast = off;
    return L;
}

// ------------------------------------------------------------------ tensor maps

int encode_3d(CUtensorMap* m, CUtensorMapDataType dt, int esize, const void* base, uint64_t d, uint64_t rows,
              uint64_t planes, uint32_t box_x, const char* name,
              CUtensorMapSwizzle swizzle = CU_TENSOR_MAP_SWIZZLE_128B, uint32_t box_rows = lca::kTileRows) {
    EncodeTiledFn enc = get_encode_fn();
    if (enc == nullptr) return fail(LCA_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable from the driver");
    cuuint64_t dims[3] = {d, rows, planes};
    cuuint64_t strides[2] = {d * (uint64_t)esize, d * rows * (uint64_t)esize};
    cuuint32_t box[3] = {box_x, box_rows, 1};
    cuuint32_t estr[3] = {1, 1, 1};
    CUresult r = enc(m, dt, 3, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                     swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(LCA_ERR_CUDA, "cuTensorMapEncodeTiled(%s) failed with CUresult %d", name, (int)r);
    return LCA_OK;
}

// Token-major tensor [batch][n][heads][d] as the 4-D map {d, heads, n, batch} (strides in
// increasing order), box box_x columns x 1 head x 128 rows x 1 batch: the box lands in shared
// memory like a box_x x 128 box of a head-major tensor.
int encode_tok(CUtensorMap* m, CUtensorMapDataType dt, int esize, const void* base, uint64_t d, uint64_t heads,
               uint64_t rows, uint64_t batch, uint32_t box_x, const char* name,
               CUtensorMapSwizzle swizzle = CU_TENSOR_MAP_SWIZZLE_128B) {
    EncodeTiledFn enc = get_encode_fn();
    if (enc == nullptr) return fail(LCA_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable from the driver");
    cuuint64_t dims[4] = {d, heads, rows, batch};
    cuuint64_t strides[3] = {d * (uint64_t)esize, heads * d * (uint64_t)esize, rows * heads * d * (uint64_t)esize};
    cuuint32_t box[4] = {box_x, 1, (cuuint32_t)lca::kTileRows, 1};
    cuuint32_t estr[4] = {1, 1, 1, 1};
    CUresult r = enc(m, dt, 4, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                     swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(LCA_ERR_CUDA, "cuTensorMapEncodeTiled(%s) failed with CUresult %d", name, (int)r);
    return LCA_OK;
}

// Compact global rows [G][3][bh][d] (16-bit): dims {d, bh, G} with the row stride of a
// whole compact row, box 64 columns x 1 head x 128 rows (lands in shared memory exactly
// like a 64 x 128 box of a [bh][n][d] tensor).
int encode_compact(CUtensorMap* m, CUtensorMapDataType dt, const void* base, uint64_t d, uint64_t bh, uint64_t G,
                   const char* name, uint64_t planes_per_row = 3, uint32_t box_rows = lca::kTileRows) {
    EncodeTiledFn enc = get_encode_fn();
    if (enc == nullptr) return fail(LCA_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable from the driver");
    cuuint64_t dims[3] = {d, bh, G};
    cuuint64_t strides[2] = {d * 2, planes_per_row * bh * d * 2};
    cuuint32_t box[3] = {64, 1, box_rows};
    cuuint32_t estr[3] = {1, 1, 1};
    CUresult r = enc(m, dt, 3, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                     CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(LCA_ERR_CUDA, "cuTensorMapEncodeTiled(%s) failed with CUresult %d", name, (int)r);
    return LCA_OK;
}

unsigned long long wait_timeout_ns() {
    static unsigned long long v = [] {
        const char* s = getenv("LCA_WAIT_TIMEOUT_MS");
        long long ms = s ? atoll(s) : 2000;
        if (ms <= 0) ms = 2000;
        return (unsigned long long)ms * 1000000ull;
    }();
    return v;
}

}  // namespace

int lca::device_info(int** err_word, unsigned long long* wait_ns) {
    int dev = 0;
    const int st = check_device(&dev, err_word);
    if (st != LCA_OK) return st;
    *wait_ns = wait_timeout_ns();
    return LCA_OK;
}

namespace {

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int check_workspace(const Layout& L, void* workspace, size_t workspace_bytes) {
    if (workspace_bytes < L.total)
        return fail(LCA_ERR_WORKSPACE, "workspace needs %zu bytes, got %zu", L.total, workspace_bytes);
    if (L.total > 0 && (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) % 256) != 0))
        return fail(LCA_ERR_WORKSPACE, "workspace must be non-NULL and 256-byte aligned");
    return LCA_OK;
}

int check_io(const void* q, const void* k, const void* v, const void* out, const float* lse) {
    if (q == nullptr || k == nullptr || v == nullptr || out == nullptr)
        return fail(LCA_ERR_INVALID_ARGUMENT, "q, k, v and out must be non-NULL");
    if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out))
        return fail(LCA_ERR_INVALID_ARGUMENT, "q, k, v and out must be 16-byte aligned");
    if (lse != nullptr && (reinterpret_cast<uintptr_t>(lse) & 3u))
        return fail(LCA_ERR_INVALID_ARGUMENT, "lse must be 4-byte aligned");
    return LCA_OK;
}

// ------------------------------------------------------------------ launch steps

// Compact copies of the global rows this problem's Q / K / V hold (zeros for global rows
// owned by other shards) and the sorted index list.
int enqueue_gather(const Problem& P, const Layout& L, const void* q, const void* k, const void* v, uint8_t* ws,
                   cudaStream_t stream) {
    if (P.G == 0) return LCA_OK;
    static thread_local lca::GatherParams gp;
    uint8_t* qg = ws + L.off_globals;
    for (int first = 0; first < (int)P.G; first += lca::kGatherChunk) {
        gp.n = (int)P.n;
        gp.q_off = (int)P.q_off;
        gp.heads = (int)P.heads;
        gp.s_b = P.s_b();
        gp.s_h = P.s_h();
        gp.s_n = P.s_n();
        gp.num_global = (int)P.G;
        gp.bh = (int)P.bh;
        gp.first = first;
        gp.count = std::min<int>(lca::kGatherChunk, (int)P.G - first);
        gp.gidx_out = reinterpret_cast<int*>(ws + L.off_gidx);
        gp.compact = reinterpret_cast<uint16_t*>(qg);
        for (int i = 0; i < gp.count; ++i) gp.idx[i] = P.gl[(size_t)first + i];
        cudaError_t e = lca::launch_gather((int)P.d, q, k, v, gp, (int)P.bh, stream);
        if (e != cudaSuccess) return fail_cuda(e, "gather launch");
    }
    return LCA_OK;
}

// The main kernel over band and global-row units.
// fp16 copy of V (the optional workspace suffix): this rank's V rows, the compact global V
// rows (complete once gathered, and for a shard once exchanged) and the received halos.
// Zeroes the words of the optional suffix that a forward starts from: the work-unit counter
// and, with the fp16 copy of V, the word beside it that records a failed conversion.
int clear_suffix_words(const Layout& L, uint8_t* ws, bool v16, cudaStream_t stream) {
    cudaError_t e = v16 ? cudaMemsetAsync(ws + L.off_v16bad, 0, 2 * sizeof(int), stream)
                        : cudaMemsetAsync(ws + L.off_counter, 0, sizeof(unsigned int), stream);
    return e == cudaSuccess ? LCA_OK : fail_cuda(e, "workspace word reset");
}

// `clear`: zero the words first (else the caller has, earlier on the stream).
int enqueue_convert_v16(const Problem& P, const Layout& L, const void* v, uint8_t* ws, cudaStream_t stream,
                        bool clear = true) {
    lca::ConvertParams cv;
    memset(&cv, 0, sizeof(cv));
    const long long d = P.d, bh = P.bh;
    auto add = [&](const uint16_t* src, uint16_t* dst, long long planes, long long rows, long long src_plane,
                   long long src_row, long long dst_plane, long long dst_row) {
        lca::ConvertSegment& g = cv.seg[cv.n_segments++];
        g.src = src;
        g.dst = dst;
        g.planes = (int)planes;
        g.rows = (int)rows;
        g.src_plane = src_plane;
        g.src_row = src_row;
        g.dst_plane = dst_plane;
        g.dst_row = dst_row;
        g.heads = 1;
        g.src_head = 0;
    };
    add(static_cast<const uint16_t*>(v), reinterpret_cast<uint16_t*>(ws + L.off_v16), bh, P.n, P.s_b(), P.s_n(), P.n * d,
        d);
    cv.seg[0].heads = (int)P.heads;  // the caller's V in its own layout
    cv.seg[0].src_head = P.s_h();
    if (P.G > 0) {
        // compact rows [G][3][bh][d]: the v plane of row g starts 2 * bh * d elements in
        const uint16_t* vg = reinterpret_cast<const uint16_t*>(ws + L.off_globals) + 2 * bh * d;
        add(vg, reinterpret_cast<uint16_t*>(ws + L.off_vg16), bh, P.G, d, 3 * bh * d, d, bh * d);
    }
    if (L.halo_block > 0) {
        // receive blocks [2 sides][2 (k, v)][bh][halo][d]: the V planes of side s
        const long long halo = P.halo(), plane = halo * d;
        for (int side = 0; side < 2; ++side) {
            const size_t off = ((size_t)(2 * side + 1) * bh) * plane * 2;
            add(reinterpret_cast<const uint16_t*>(ws + L.off_recv + off), reinterpret_cast<uint16_t*>(ws + L.off_vh16 + off),
                bh, halo, plane, d, plane, d);
        }
    }
    cv.any_bad = reinterpret_cast<int*>(ws + L.off_v16bad);
    int st;
    if (clear && (st = clear_suffix_words(L, ws, true, stream)) != LCA_OK) return st;
    cudaError_t e = lca::launch_convert_v16((int)P.d, cv, stream);
    if (e != cudaSuccess) return fail_cuda(e, "fp16 V copy launch");
    return LCA_OK;
}

// Every tensor map of one main-kernel launch.  Maps depend only on the pointers and the
// problem's shape, so they are cached per thread (the last kMapCache call signatures): a
// caller that repeats a call -- a serving loop, a bench, a sharded step -- skips the
// encoding (up to 13 driver calls).
struct MapKey {
    const void* q;
    const void* k;
    const void* v;
    const void* out;
    const void* ws;
    int64_t n, n_total, q_off, d, bh, G, window, world;
    int dtype, out_dtype, sharded, v16, n_splits, dev, tok_major, heads;
};
constexpr int kMapCache = 4;
thread_local MapKey g_map_key[kMapCache];
thread_local lca::TensorMaps g_map_val[kMapCache];
thread_local bool g_map_ok[kMapCache];
thread_local int g_map_next = 0;

int encode_maps(const Problem& P, const Layout& L, const void* q, const void* k, const void* v, void* out,
                uint8_t* ws, bool v16, lca::TensorMaps& tm) {
    const bool bf16 = P.dtype == LCA_DTYPE_BF16;
    const CUtensorMapDataType tdt = bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const int n = (int)P.n;
    const int d = (int)P.d;
    const uint64_t bh = (uint64_t)P.bh;
    const int halo = (int)P.halo();
    int st;
    memset(&tm, 0, sizeof(tm));
    const CUtensorMapDataType odt = P.out_dtype == LCA_DTYPE_F32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                    : P.out_dtype == LCA_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                                    : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const int osize = P.out_dtype == LCA_DTYPE_F32 ? 4 : 2;
    // fp32 output in 32-column boxes of 128-byte swizzled rows; 16-bit output in 32-column
    // boxes of 64-byte rows, unswizzled
    const CUtensorMapSwizzle osw = P.out_dtype == LCA_DTYPE_F32 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE;
    if (P.tok_major) {
        const uint64_t H = (uint64_t)P.heads, B = bh / H;
        if ((st = encode_tok(&tm.q, tdt, 2, q, d, H, n, B, 64, "q")) != LCA_OK) return st;
        if ((st = encode_tok(&tm.k, tdt, 2, k, d, H, n, B, 64, "k")) != LCA_OK) return st;
        if ((st = encode_tok(&tm.v, tdt, 2, v, d, H, n, B, 64, "v")) != LCA_OK) return st;
        if ((st = encode_tok(&tm.o, odt, osize, out, d, H, n, B, 32, "out", osw)) != LCA_OK) return st;
    } else {
        if ((st = encode_3d(&tm.q, tdt, 2, q, d, n, bh, 64, "q")) != LCA_OK) return st;
        if ((st = encode_3d(&tm.k, tdt, 2, k, d, n, bh, 64, "k")) != LCA_OK) return st;
        if ((st = encode_3d(&tm.v, tdt, 2, v, d, n, bh, 64, "v")) != LCA_OK) return st;
        if ((st = encode_3d(&tm.o, odt, osize, out, d, n, bh, 32, "out", osw)) != LCA_OK) return st;
    }
    if (halo > 0) {
        // recv block [2 sides][2 (k, v)][bh][halo][d]: K planes at z = side * 2bh + b from
        // the block start, V planes the same from bh planes further on
        uint8_t* recv = ws + L.off_recv;
        const size_t plane = (size_t)halo * d * 2;
        if ((st = encode_3d(&tm.kh, tdt, 2, recv, d, halo, 4 * bh, 64, "k_halo")) != LCA_OK) return st;
        if ((st = encode_3d(&tm.vh, tdt, 2, recv + bh * plane, d, halo, 3 * bh, 64, "v_halo")) != LCA_OK) return st;
    } else {
        tm.kh = tm.k;
        tm.vh = tm.v;
    }
    if (P.G > 0) {
        uint8_t* qg = ws + L.off_globals;
        const uint64_t G = (uint64_t)P.G;
        const size_t plane = (size_t)bh * d * 2;  // one of q / k / v within a compact row
        if ((st = encode_compact(&tm.qg, tdt, qg, d, bh, G, "q_global")) != LCA_OK) return st;
        if ((st = encode_compact(&tm.kg, tdt, qg + plane, d, bh, G, "k_global")) != LCA_OK) return st;
        if ((st = encode_compact(&tm.vg, tdt, qg + 2 * plane, d, bh, G, "v_global")) != LCA_OK) return st;
        if ((st = encode_3d(&tm.po, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, ws + L.off_po, d, G,
                            (uint64_t)2 * L.n_splits * bh, 32, "partial_out")) != LCA_OK)
            return st;
    } else {
        // unused maps still need valid encodings for the kernel parameter block
        tm.qg = tm.q;
        tm.kg = tm.k;
        tm.vg = tm.v;
        tm.po = tm.q;
    }
    tm.v16 = tm.v;
    tm.vg16 = tm.vg;
    tm.vh16 = tm.vh;
    if (v16) {
        if (halo > 0) {
            const size_t plane = (size_t)halo * d * 2;
            if ((st = encode_3d(&tm.vh16, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, ws + L.off_vh16 + bh * plane, d, halo,
                                3 * bh, 64, "v_halo_fp16")) != LCA_OK)
                return st;
        }
        const CUtensorMapDataType f16 = CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
        if ((st = encode_3d(&tm.v16, f16, 2, ws + L.off_v16, d, n, bh, 64, "v_fp16")) != LCA_OK) return st;
        if (P.G > 0 &&
            (st = encode_compact(&tm.vg16, f16, ws + L.off_vg16, d, bh, (uint64_t)P.G, "v_global_fp16", 1)) != LCA_OK)
            return st;
    }
    return LCA_OK;
}

int cached_maps(const Problem& P, const Layout& L, int dev, const void* q, const void* k, const void* v, void* out,
                uint8_t* ws, bool v16, lca::TensorMaps& tm) {
    MapKey key;
    memset(&key, 0, sizeof(key));  // padding too: keys are compared bytewise
    key.q = q;
    key.k = k;
    key.v = v;
    key.out = out;
    key.ws = ws;
    key.n = P.n;
    key.n_total = P.n_total;
    key.q_off = P.q_off;
    key.d = P.d;
    key.bh = P.bh;
    key.G = P.G;
    key.window = P.window;
    key.world = P.world;
    key.dtype = P.dtype;
    key.out_dtype = P.out_dtype;
    key.tok_major = P.tok_major ? 1 : 0;
    key.heads = (int)P.heads;
    key.sharded = P.sharded ? 1 : 0;
    key.v16 = v16 ? 1 : 0;
    key.n_splits = L.n_splits;
    key.dev = dev;
    for (int i = 0; i < kMapCache; ++i) {
        if (g_map_ok[i] && memcmp(&g_map_key[i], &key, sizeof(key)) == 0) {
            tm = g_map_val[i];
            return LCA_OK;
        }
    }
    const int st = encode_maps(P, L, q, k, v, out, ws, v16, tm);
    if (st != LCA_OK) return st;
    const int slot = g_map_next;
    g_map_next = (g_map_next + 1) % kMapCache;
    g_map_key[slot] = key;
    g_map_val[slot] = tm;
    g_map_ok[slot] = true;
    return LCA_OK;
}

int enqueue_main(const Problem& P, const Layout& L, int dev, int* err_word, const void* q, const void* k,
                 const void* v, void* out, float* lse, uint8_t* ws, cudaStream_t stream, bool v16 = false,
                 bool dynamic_units = false, bool clear_counter = true) {
    const bool bf16 = P.dtype == LCA_DTYPE_BF16;
    const int n = (int)P.n;
    const int d = (int)P.d;
    int st;
    lca::TensorMaps tm;
    if ((st = cached_maps(P, L, dev, q, k, v, out, ws, v16, tm)) != LCA_OK) return st;

    lca::MainParams p;
    memset(&p, 0, sizeof(p));
    p.n = n;
    p.q_off = (int)P.q_off;
    p.n_total = (int)P.n_total;
    p.sharded = P.sharded ? 1 : 0;
    p.halo = (int)P.halo();
    p.bh = (int)P.bh;
    p.window = (int)P.window;
    p.lead = (int)P.lead();
    p.key_lo = (int)std::max<int64_t>(0, P.q_off - P.window);
    p.key_hi = (int)std::min<int64_t>(P.n_total, P.q_off + P.n + P.window);
    if (!P.sharded) {
        p.key_lo = 0;
        p.key_hi = n;
    }
    p.gk_lo = (int)P.q_off;
    p.gk_n = n;
    p.q_tiles = (n + lca::kTileRows - 1) / lca::kTileRows;
    p.num_global = (int)P.G;
    p.scale_log2 = P.scale * 1.4426950408889634f;
    // scale == 0 gives every visible key the same weight; a tiny positive factor keeps
    // that (scores * 1e-30 round to 0 in the exponent) while masked scores stay -inf.
    if (p.scale_log2 == 0.f) p.scale_log2 = 1e-30f;
    p.lse = lse;
    p.err = err_word;
    p.timeout_ns = wait_timeout_ns();
    p.out16 = P.out_dtype == LCA_DTYPE_F32 ? 0 : (P.out_dtype == LCA_DTYPE_BF16 ? lca::kOut16BF16 : lca::kOut16F16);
    p.causal = P.causal ? 1 : 0;
    p.n_head_windows = (int)P.head_window.size();
    for (size_t h = 0; h < P.head_window.size(); ++h) p.head_window[h] = P.head_window[h];
    p.heads4d = P.tok_major ? (int)P.heads : 0;
    p.seg_mode = P.seg_mode;
    p.seg_len = (int)P.seg_len;
    p.n_segs = P.seg_start.empty() ? 0 : (int)P.seg_start.size() - 1;
    for (size_t i = 0; i < P.seg_start.size(); ++i) p.seg_start[i] = P.seg_start[i];
    if (P.G > 0) {
        p.g_tiles = L.g_tiles;
        p.n_splits = L.n_splits;
        p.split_tiles = L.split_tiles;
        p.n_grow_units = (int)(P.bh * L.g_tiles * L.n_splits);
        p.gidx = reinterpret_cast<const int*>(ws + L.off_gidx);
        p.part_lse = reinterpret_cast<float*>(ws + L.off_plse);
    }
    if (v16) p.v16_bad = reinterpret_cast<const int*>(ws + L.off_v16bad);

    p.q_pairs = (p.q_tiles + 1) / 2;
    const long long units = (long long)p.n_grow_units + (long long)P.bh * p.q_pairs;
    if (units > INT_MAX) return fail(LCA_ERR_UNSUPPORTED, "problem too large (%lld work units)", units);
    p.n_band_units = (int)(P.bh * p.q_pairs);
    // key-tile steps of one unit of each kind: the longer kind is handed out first
    const int64_t band_steps = 2 * ((P.lead() + P.window + 2 * lca::kTileRows - 1) / lca::kTileRows + p.g_tiles);
    p.grow_first = (P.G > 0 && (int64_t)p.split_tiles >= band_steps) ? 1 : 0;
    const int grid = (int)std::min<long long>(units, g_dev_sms[dev]);
    if (dynamic_units) {
        p.unit_counter = reinterpret_cast<unsigned int*>(ws + L.off_counter);
        // (with the fp16 copy of V, the copy's memset cleared it)
        if (!v16 && clear_counter && (st = clear_suffix_words(L, ws, false, stream)) != LCA_OK) return st;
    }
    const bool timed = g_ev_before_main != nullptr && g_ev_after_main != nullptr;
    cudaError_t e;
    if (timed && (e = cudaEventRecord(g_ev_before_main, stream)) != cudaSuccess)
        return fail_cuda(e, "timing event record");
    e = lca::launch_main(d, bf16, tm, p, grid, stream, v16);
    if (e != cudaSuccess) return fail_cuda(e, "main kernel launch");
    if (timed && (e = cudaEventRecord(g_ev_after_main, stream)) != cudaSuccess)
        return fail_cuda(e, "timing event record");
    return LCA_OK;
}

// Merge of the main kernel's global-row partials: over the rows of out / lse, or (for a
// shard) into this shard's packed row partial.
int enqueue_combine_splits(const Problem& P, const Layout& L, void* out, float* lse, uint8_t* ws,
                           cudaStream_t stream) {
    if (P.G == 0) return LCA_OK;
    lca::CombineParams cp;
    memset(&cp, 0, sizeof(cp));
    cp.bh = (int)P.bh;
    cp.num_global = (int)P.G;
    cp.n_parts = 2 * L.n_splits;
    cp.split_tiles = L.split_tiles;
    cp.split_keys = (int)P.n;
    cp.part_stride_o = (size_t)P.bh * P.G * P.d;
    cp.part_stride_lse = (size_t)P.bh * P.G;
    cp.part_o = reinterpret_cast<const float*>(ws + L.off_po);
    cp.part_lse = reinterpret_cast<const float*>(ws + L.off_plse);
    cp.gidx = reinterpret_cast<const int*>(ws + L.off_gidx);
    if (P.sharded) {
        cp.out_o = reinterpret_cast<float*>(ws + L.off_rowpart);
        cp.out_lse = cp.out_o + (size_t)P.bh * P.G * P.d;
    } else {
        cp.o = out;
        cp.lse = lse;
        cp.out16 = P.out_dtype == LCA_DTYPE_F32 ? 0 : (P.out_dtype == LCA_DTYPE_BF16 ? lca::kOut16BF16 : lca::kOut16F16);
        cp.n_rows = (int)P.n;
        cp.row_off = 0;
        cp.heads = (int)P.heads;
        cp.o_b = P.s_b();
        cp.o_h = P.s_h();
        cp.o_n = P.s_n();
    }
    cudaError_t e = lca::launch_combine((int)P.d, cp, stream);
    if (e != cudaSuccess) return fail_cuda(e, "combine launch");
    return LCA_OK;
}

int run_problem(const Problem& P, const void* q, const void* k, const void* v, void* out, float* lse, void* workspace,
                size_t workspace_bytes, void* stream_ptr);

int check_out_flags(int out_dtype, int flags) {
    if (out_dtype != LCA_DTYPE_F32 && out_dtype != LCA_DTYPE_F16 && out_dtype != LCA_DTYPE_BF16)
        return fail(LCA_ERR_UNSUPPORTED, "out_dtype %d is not supported (fp32, fp16 or bf16)", out_dtype);
    if ((flags & ~(LCA_FLAG_CAUSAL | LCA_FLAG_TOKEN_MAJOR)) != 0)
        return fail(LCA_ERR_INVALID_ARGUMENT, "unknown flags 0x%x", flags);
    return LCA_OK;
}

// One radius per head: the largest becomes *window_size (it sizes the workspace); the
// per-head list is kept unless all radii are equal.
int parse_head_windows(int64_t heads, int64_t seq_len, const int64_t* head_window_sizes, int64_t* window_size,
                       std::vector<int>& out) {
    out.clear();
    if (head_window_sizes == nullptr) return LCA_OK;
    if (heads > LCA_MAX_HEAD_WINDOWS)
        return fail(LCA_ERR_UNSUPPORTED, "radii of their own for %lld heads (at most %d)", (long long)heads,
                    LCA_MAX_HEAD_WINDOWS);
    int64_t wmax = 0;
    bool uniform = true;
    for (int64_t h = 0; h < heads; ++h) {
        if (head_window_sizes[h] < 0)
            return fail(LCA_ERR_INVALID_ARGUMENT, "head_window_sizes[%lld] = %lld must be >= 0", (long long)h,
                        (long long)head_window_sizes[h]);
        wmax = std::max(wmax, head_window_sizes[h]);
        uniform = uniform && head_window_sizes[h] == head_window_sizes[0];
    }
    *window_size = wmax;
    if (!uniform)
        for (int64_t h = 0; h < heads; ++h) out.push_back((int)std::min(head_window_sizes[h], seq_len));
    return LCA_OK;
}

}  // namespace

// ====================================================================== C ABI

extern "C" {

int lca_abi_version(void) { return LCA_ABI_VERSION; }

const char* lca_status_string(int status) {
    switch (status) {
        case LCA_OK: return "ok";
        case LCA_ERR_INVALID_ARGUMENT: return "invalid argument";
        case LCA_ERR_INDEX: return "global token index out of range";
        case LCA_ERR_UNSUPPORTED: return "unsupported configuration";
        case LCA_ERR_WORKSPACE: return "workspace too small or misaligned";
        case LCA_ERR_CUDA: return "CUDA error";
        case LCA_ERR_DEVICE: return "device-side error";
        default: return "unknown status";
    }
}

const char* lca_last_error(void) { return g_last_error.c_str(); }

int lca_normalize_global_tokens(const int64_t* tokens, int64_t count, int64_t seq_len, int32_t* out,
                                int64_t* out_count) {
    if (out_count == nullptr) return fail(LCA_ERR_INVALID_ARGUMENT, "out_count is NULL");
    if (count < 0) return fail(LCA_ERR_INVALID_ARGUMENT, "negative global token count %lld", (long long)count);
    if (count > 0 && (tokens == nullptr || out == nullptr))
        return fail(LCA_ERR_INVALID_ARGUMENT, "global token arrays are NULL");
    if (seq_len < 0 || seq_len > INT_MAX) return fail(LCA_ERR_INVALID_ARGUMENT, "seq_len %lld out of range", (long long)seq_len);
    std::vector<int32_t> v;
    v.reserve((size_t)count);
    for (int64_t i = 0; i < count; ++i) {
        int64_t t = tokens[i];
        if (t < -seq_len || t >= seq_len)
            return fail(LCA_ERR_INDEX, "index %lld is out of bounds for dimension 0 with size %lld", (long long)t,
                        (long long)seq_len);
        if (t < 0) t += seq_len;
        v.push_back((int32_t)t);
    }
    std::sort(v.begin(), v.end());
    v.erase(std::unique(v.begin(), v.end()), v.end());
    std::copy(v.begin(), v.end(), out);
    *out_count = (int64_t)v.size();
    return LCA_OK;
}

}  // extern "C"

namespace lca {
int workspace_bytes(int64_t batch, int64_t heads, int64_t seq_len, int64_t head_dim, int64_t window_size,
                    int64_t num_unique_global, int dtype, bool with_fp16_v, size_t* out_bytes) {
    if (out_bytes == nullptr) return fail(LCA_ERR_INVALID_ARGUMENT, "out_bytes is NULL");
    if (batch < 0 || heads < 0 || seq_len < 0 || num_unique_global < 0)
        return fail(LCA_ERR_INVALID_ARGUMENT, "negative size");
    int st = check_dtype_dim(dtype, head_dim);
    if (st != LCA_OK) return st;
    if (window_size < 0) return fail(LCA_ERR_INVALID_ARGUMENT, "window_size must be >= 0");
    Problem P;
    P.bh = batch * heads;
    P.n_total = P.n = seq_len;
    P.d = head_dim;
    P.window = std::min(window_size, seq_len);
    P.G = std::min(num_unique_global, seq_len);
    P.dtype = dtype;
    const Layout L = make_layout(P);
    *out_bytes = with_fp16_v ? L.total_fast : L.total;
    return LCA_OK;
}
}  // namespace lca

extern "C" {

int lca_swa_workspace_size(int64_t batch, int64_t heads, int64_t seq_len, int64_t head_dim, int64_t window_size,
                           int64_t num_unique_global, int dtype, size_t* out_bytes) {
    return lca::workspace_bytes(batch, heads, seq_len, head_dim, window_size, num_unique_global, dtype, true,
                                out_bytes);
}

int lca_swa_forward(const void* q, const void* k, const void* v, float* out, float* lse, int dtype,
                    int64_t batch, int64_t heads, int64_t seq_len, int64_t head_dim, int64_t window_size,
                    float scale, const int64_t* global_tokens, int64_t num_global_tokens, void* workspace,
                    size_t workspace_bytes, void* stream_ptr) {
    return lca_swa_forward_ex(q, k, v, out, LCA_DTYPE_F32, lse, dtype, batch, heads, seq_len, head_dim, window_size,
                              nullptr, scale, 0, global_tokens, num_global_tokens, workspace, workspace_bytes,
                              stream_ptr);
}

int lca_swa_forward_ex(const void* q, const void* k, const void* v, void* out, int out_dtype, float* lse, int dtype,
                       int64_t batch, int64_t heads, int64_t seq_len, int64_t head_dim, int64_t window_size,
                       const int64_t* head_window_sizes, float scale, int flags, const int64_t* global_tokens,
                       int64_t num_global_tokens, void* workspace, size_t workspace_bytes, void* stream_ptr) {
    g_last_error.clear();
    int st = check_out_flags(out_dtype, flags);
    if (st != LCA_OK) return st;
    std::vector<int> head_window;
    st = parse_head_windows(heads, seq_len, head_window_sizes, &window_size, head_window);
    if (st != LCA_OK) return st;
    Problem P;
    st = parse_common(P, dtype, batch, heads, seq_len, head_dim, window_size, scale, global_tokens,
                      num_global_tokens);
    if (st != LCA_OK) return st;
    P.head_window = std::move(head_window);
    P.out_dtype = out_dtype;
    P.causal = (flags & LCA_FLAG_CAUSAL) != 0;
    P.tok_major = (flags & LCA_FLAG_TOKEN_MAJOR) != 0;
    return run_problem(P, q, k, v, out, lse, workspace, workspace_bytes, stream_ptr);
}

// ------------------------------------------------------------------ packed sequences

int lca_swa_forward_varlen(const void* q, const void* k, const void* v, void* out, int out_dtype, float* lse,
                           int dtype, int64_t heads, int64_t total_len, int64_t head_dim, int64_t window_size,
                           const int64_t* head_window_sizes, float scale, int flags, const int64_t* cu_seqlens,
                           int64_t num_seqs, const int64_t* global_tokens, int64_t num_global_tokens,
                           void* workspace, size_t workspace_bytes, void* stream_ptr) {
    g_last_error.clear();
    int st = check_out_flags(out_dtype, flags);
    if (st != LCA_OK) return st;
    if (cu_seqlens == nullptr || num_seqs < 1)
        return fail(LCA_ERR_INVALID_ARGUMENT, "cu_seqlens needs num_seqs + 1 >= 2 offsets");
    if (num_seqs > LCA_MAX_SEQUENCES)
        return fail(LCA_ERR_UNSUPPORTED, "%lld sequences in one call (at most %d)", (long long)num_seqs,
                    LCA_MAX_SEQUENCES);
    if (cu_seqlens[0] != 0 || cu_seqlens[num_seqs] != total_len)
        return fail(LCA_ERR_INVALID_ARGUMENT, "cu_seqlens must run from 0 to total_len (%lld)", (long long)total_len);
    for (int64_t i = 0; i < num_seqs; ++i)
        if (cu_seqlens[i + 1] < cu_seqlens[i])
            return fail(LCA_ERR_INVALID_ARGUMENT, "cu_seqlens must not decrease (at %lld)", (long long)i);
    if (num_global_tokens < 0 || (num_global_tokens > 0 && global_tokens == nullptr))
        return fail(LCA_ERR_INVALID_ARGUMENT, "bad global token list");
    std::vector<int> head_window;
    if ((st = parse_head_windows(heads, total_len, head_window_sizes, &window_size, head_window)) != LCA_OK)
        return st;
    Problem P;
    if ((st = parse_common(P, dtype, 1, heads, total_len, head_dim, window_size, scale, nullptr, 0)) != LCA_OK)
        return st;
    // the token list applies to every non-empty sequence, indexed within it the way the
    // reference indexes one sequence (negative from its end; outside it is an error)
    std::vector<int32_t> norm((size_t)num_global_tokens + 1);
    for (int64_t sq = 0; sq < num_seqs; ++sq) {
        const int64_t len = cu_seqlens[sq + 1] - cu_seqlens[sq];
        if (len == 0 || num_global_tokens == 0) continue;
        int64_t G = 0;
        if ((st = lca_normalize_global_tokens(global_tokens, num_global_tokens, len, norm.data(), &G)) != LCA_OK) {
            const std::string why = lca_last_error();
            return fail(st, "sequence %lld (length %lld): %s", (long long)sq, (long long)len, why.c_str());
        }
        for (int64_t i = 0; i < G; ++i) P.gl.push_back((int32_t)(cu_seqlens[sq] + norm[(size_t)i]));
    }
    std::sort(P.gl.begin(), P.gl.end());
    P.G = (int64_t)P.gl.size();
    P.head_window = std::move(head_window);
    P.out_dtype = out_dtype;
    P.causal = (flags & LCA_FLAG_CAUSAL) != 0;
    P.tok_major = (flags & LCA_FLAG_TOKEN_MAJOR) != 0;
    if (num_seqs > 1) {
        P.seg_mode = lca::kSegVarlen;
        for (int64_t i = 0; i <= num_seqs; ++i) P.seg_start.push_back((int)cu_seqlens[i]);
    }
    return run_problem(P, q, k, v, out, lse, workspace, workspace_bytes, stream_ptr);
}

// ------------------------------------------------------------------ dilated windows

}  // extern "C"

namespace {

// Bytes of the residue-order copies a dilated forward keeps ahead of the problem's own
// workspace: Q, K, V, O and LSE, each region 1024-byte aligned.
size_t dilated_prefix_bytes(int64_t bh, int64_t n, int64_t d, int out_dtype) {
    const size_t plane = (size_t)bh * n * d;
    const size_t osize = out_dtype == LCA_DTYPE_F32 ? 4 : 2;
    return 3 * align_up(plane * 2, kAlign) + align_up(plane * osize, kAlign) + align_up((size_t)bh * n * 4, kAlign);
}

int permute(const void* src, void* dst, int64_t planes, int64_t n, int64_t dil, int64_t row_bytes, bool to_residue,
            cudaStream_t stream) {
    lca::PermuteParams pp;
    pp.src = static_cast<const uint8_t*>(src);
    pp.dst = static_cast<uint8_t*>(dst);
    pp.planes = planes;
    pp.n = (int)n;
    pp.dil = (int)dil;
    pp.row_bytes = (int)row_bytes;
    pp.to_residue = to_residue ? 1 : 0;
    cudaError_t e = lca::launch_permute_rows(pp, stream);
    if (e != cudaSuccess) return fail_cuda(e, "residue-order copy launch");
    return LCA_OK;
}

}  // namespace

extern "C" {

int lca_swa_dilated_workspace_size(int64_t batch, int64_t heads, int64_t seq_len, int64_t head_dim,
                                   int64_t window_size, int64_t dilation, int64_t num_unique_global, int dtype,
                                   int out_dtype, size_t* out_bytes) {
    if (out_bytes == nullptr) return fail(LCA_ERR_INVALID_ARGUMENT, "out_bytes is NULL");
    if (dilation < 1) return fail(LCA_ERR_INVALID_ARGUMENT, "dilation must be >= 1");
    int st = check_out_flags(out_dtype, 0);
    if (st != LCA_OK) return st;
    size_t inner = 0;
    if ((st = lca::workspace_bytes(batch, heads, seq_len, head_dim, window_size, num_unique_global, dtype, true,
                                   &inner)) != LCA_OK)
        return st;
    *out_bytes = dilation == 1 ? inner : dilated_prefix_bytes(batch * heads, seq_len, head_dim, out_dtype) + inner;
    return LCA_OK;
}

int lca_swa_forward_dilated(const void* q, const void* k, const void* v, void* out, int out_dtype, float* lse,
                            int dtype, int64_t batch, int64_t heads, int64_t seq_len, int64_t head_dim,
                            int64_t window_size, const int64_t* head_window_sizes, int64_t dilation, float scale,
                            int flags, const int64_t* global_tokens, int64_t num_global_tokens, void* workspace,
                            size_t workspace_bytes, void* stream_ptr) {
    g_last_error.clear();
    if (dilation < 1) return fail(LCA_ERR_INVALID_ARGUMENT, "dilation must be >= 1 (got %lld)", (long long)dilation);
    if (dilation == 1)
        return lca_swa_forward_ex(q, k, v, out, out_dtype, lse, dtype, batch, heads, seq_len, head_dim, window_size,
                                  head_window_sizes, scale, flags, global_tokens, num_global_tokens, workspace,
                                  workspace_bytes, stream_ptr);
    int st = check_out_flags(out_dtype, flags);
    if (st != LCA_OK) return st;
    if (flags & LCA_FLAG_CAUSAL)
        return fail(LCA_ERR_UNSUPPORTED, "the causal variant has no dilated form in this build");
    if (flags & LCA_FLAG_TOKEN_MAJOR)
        return fail(LCA_ERR_UNSUPPORTED, "the dilated window takes head-major tensors in this build");
    if (seq_len % dilation != 0)
        return fail(LCA_ERR_UNSUPPORTED, "seq_len %lld is not a multiple of the dilation %lld", (long long)seq_len,
                    (long long)dilation);
    std::vector<int> head_window;
    if ((st = parse_head_windows(heads, seq_len, head_window_sizes, &window_size, head_window)) != LCA_OK) return st;
    Problem P;
    if ((st = parse_common(P, dtype, batch, heads, seq_len, head_dim, window_size, scale, global_tokens,
                           num_global_tokens)) != LCA_OK)
        return st;
    if (P.bh == 0 || P.n == 0) return LCA_OK;
    if ((st = check_io(q, k, v, out, lse)) != LCA_OK) return st;
    // The band of row i = r + dilation * t (residue r) is the keys r + dilation * t' with
    // |t - t'| <= w: in residue order (row r * m + t, m = n / dilation) that is an ordinary
    // band of radius w inside segment r of m tokens.  Global tokens move to their residue-order
    // positions and keep seeing, and being seen by, every row.
    const int64_t m = seq_len / dilation;
    for (auto& g : P.gl) g = (int32_t)((g % dilation) * m + g / dilation);
    std::sort(P.gl.begin(), P.gl.end());
    P.head_window = std::move(head_window);
    P.out_dtype = out_dtype;
    P.seg_mode = lca::kSegEqual;
    P.seg_len = m;
    const size_t prefix = dilated_prefix_bytes(P.bh, P.n, P.d, out_dtype);
    if (workspace == nullptr || workspace_bytes < prefix || reinterpret_cast<uintptr_t>(workspace) % 256 != 0)
        return fail(LCA_ERR_WORKSPACE, "a dilated forward needs lca_swa_dilated_workspace_size bytes, 256-byte aligned");
    cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    const size_t plane = (size_t)P.bh * P.n * P.d;
    const size_t osize = out_dtype == LCA_DTYPE_F32 ? 4 : 2;
    uint8_t* rq = ws;
    uint8_t* rk = rq + align_up(plane * 2, kAlign);
    uint8_t* rv = rk + align_up(plane * 2, kAlign);
    uint8_t* ro = rv + align_up(plane * 2, kAlign);
    float* rl = reinterpret_cast<float*>(ro + align_up(plane * osize, kAlign));
    const int64_t row = P.d * 2;
    if ((st = permute(q, rq, P.bh, P.n, dilation, row, true, stream)) != LCA_OK) return st;
    if ((st = permute(k, rk, P.bh, P.n, dilation, row, true, stream)) != LCA_OK) return st;
    if ((st = permute(v, rv, P.bh, P.n, dilation, row, true, stream)) != LCA_OK) return st;
    if ((st = run_problem(P, rq, rk, rv, ro, lse != nullptr ? rl : nullptr, ws + prefix, workspace_bytes - prefix,
                          stream_ptr)) != LCA_OK)
        return st;
    if ((st = permute(ro, out, P.bh, P.n, dilation, P.d * (int64_t)osize, false, stream)) != LCA_OK) return st;
    if (lse != nullptr && (st = permute(rl, lse, P.bh, P.n, dilation, 4, false, stream)) != LCA_OK) return st;
    return LCA_OK;
}

}  // extern "C"

namespace {

// Checks the buffers and enqueues one whole-sequence problem: gather of the global rows,
// (fp16 copy of V), the main kernel, merge of the global-row splits.
int run_problem(const Problem& P, const void* q, const void* k, const void* v, void* out, float* lse, void* workspace,
                size_t workspace_bytes, void* stream_ptr) {
    int st;
    if (P.bh == 0 || P.n == 0) return LCA_OK;  // nothing to compute
    if ((st = check_io(q, k, v, out, lse)) != LCA_OK) return st;
    int dev = 0;
    int* err_word = nullptr;
    if ((st = check_device(&dev, &err_word)) != LCA_OK) return st;
    const Layout L = make_layout(P);
    if ((st = check_workspace(L, workspace, workspace_bytes)) != LCA_OK) return st;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    // the optional suffix is there (a workspace that reports 0 required bytes may be NULL)
    const bool fast = workspace != nullptr && workspace_bytes >= L.total_fast &&
                      reinterpret_cast<uintptr_t>(workspace) % 256 == 0;
    const bool v16 = fast && L.has_v16;
    // 0. zero the suffix words, 1. gather the global rows, (2. fp16 copy of V), 3. band +
    //    global-row units, 4. merge the global-row splits.  The words are cleared first so
    //    that 1-4 are consecutive kernels, each launched to overlap the one before.
    if (fast && (st = clear_suffix_words(L, ws, v16, stream)) != LCA_OK) return st;
    if ((st = enqueue_gather(P, L, q, k, v, ws, stream)) != LCA_OK) return st;
    if (v16 && (st = enqueue_convert_v16(P, L, v, ws, stream, false)) != LCA_OK) return st;
    if ((st = enqueue_main(P, L, dev, err_word, q, k, v, out, lse, ws, stream, v16, fast, false)) != LCA_OK) return st;
    return enqueue_combine_splits(P, L, out, lse, ws, stream);
}

}  // namespace

extern "C" {

// ------------------------------------------------------------------ sequence shards

int lca_swa_shard_layout(const lca_shard_desc* desc, int64_t num_unique_global, lca_shard_layout* out) {
    if (out == nullptr) return fail(LCA_ERR_INVALID_ARGUMENT, "out is NULL");
    if (num_unique_global < 0) return fail(LCA_ERR_INVALID_ARGUMENT, "negative global count");
    Problem P;
    int st = parse_shard(P, desc, nullptr, 0);
    if (st != LCA_OK) return st;
    P.G = std::min(num_unique_global, P.n_total);
    const Layout L = make_layout(P);
    memset(out, 0, sizeof(*out));
    out->total_bytes = L.total_fast;
    out->halo_rows = P.halo();
    out->globals_offset = L.off_globals;
    out->globals_bytes = (size_t)P.G * L.grow_bytes;
    out->globals_row_bytes = L.grow_bytes;
    out->halo_send_offset = L.off_send;
    out->halo_recv_offset = L.off_recv;
    out->halo_side_bytes = L.halo_block;
    out->rowpart_offset = L.off_rowpart;
    out->rowpart_bytes = L.rowpart_bytes;
    out->rowpart_all_offset = L.off_rowpart_all;
    return LCA_OK;
}

int lca_swa_shard_prepare(const lca_shard_desc* desc, const void* q, const void* k, const void* v,
                          const int64_t* global_tokens, int64_t num_global_tokens, void* workspace,
                          size_t workspace_bytes, void* stream_ptr) {
    g_last_error.clear();
    Problem P;
    int st = parse_shard(P, desc, global_tokens, num_global_tokens);
    if (st != LCA_OK) return st;
    if (P.bh == 0) return LCA_OK;
    if (q == nullptr || k == nullptr || v == nullptr || !aligned16(q) || !aligned16(k) || !aligned16(v))
        return fail(LCA_ERR_INVALID_ARGUMENT, "q, k and v must be non-NULL and 16-byte aligned");
    int dev = 0;
    int* err_word = nullptr;
    if ((st = check_device(&dev, &err_word)) != LCA_OK) return st;
    const Layout L = make_layout(P);
    if ((st = check_workspace(L, workspace, workspace_bytes)) != LCA_OK) return st;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    if ((st = enqueue_gather(P, L, q, k, v, ws, stream)) != LCA_OK) return st;
    if (P.halo() > 0) {
        lca::HaloPackParams hp;
        hp.n = (int)P.n;
        hp.halo = (int)P.halo();
        hp.bh = (int)P.bh;
        hp.d = (int)P.d;
        hp.k = static_cast<const uint16_t*>(k);
        hp.v = static_cast<const uint16_t*>(v);
        hp.send = reinterpret_cast<uint16_t*>(ws + L.off_send);
        cudaError_t e = lca::launch_halo_pack(hp, stream);
        if (e != cudaSuccess) return fail_cuda(e, "halo pack launch");
    }
    return LCA_OK;
}

int lca_swa_shard_forward(const lca_shard_desc* desc, const void* q, const void* k, const void* v, float* out,
                          float* lse, const int64_t* global_tokens, int64_t num_global_tokens, void* workspace,
                          size_t workspace_bytes, void* stream_ptr) {
    g_last_error.clear();
    Problem P;
    int st = parse_shard(P, desc, global_tokens, num_global_tokens);
    if (st != LCA_OK) return st;
    if (P.bh == 0) return LCA_OK;
    if ((st = check_io(q, k, v, out, lse)) != LCA_OK) return st;
    int dev = 0;
    int* err_word = nullptr;
    if ((st = check_device(&dev, &err_word)) != LCA_OK) return st;
    const Layout L = make_layout(P);
    if ((st = check_workspace(L, workspace, workspace_bytes)) != LCA_OK) return st;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    // the compact global rows and the halos are complete here (after the exchange)
    // the optional suffix is there (a workspace that reports 0 required bytes may be NULL)
    const bool fast = workspace != nullptr && workspace_bytes >= L.total_fast &&
                      reinterpret_cast<uintptr_t>(workspace) % 256 == 0;
    const bool v16 = fast && L.has_v16;
    if (v16 && (st = enqueue_convert_v16(P, L, v, ws, stream)) != LCA_OK) return st;
    if ((st = enqueue_main(P, L, dev, err_word, q, k, v, out, lse, ws, stream, v16, fast)) != LCA_OK) return st;
    return enqueue_combine_splits(P, L, out, lse, ws, stream);
}

int lca_swa_shard_finish(const lca_shard_desc* desc, float* out, float* lse, const int64_t* global_tokens,
                         int64_t num_global_tokens, void* workspace, size_t workspace_bytes, void* stream_ptr) {
    g_last_error.clear();
    Problem P;
    int st = parse_shard(P, desc, global_tokens, num_global_tokens);
    if (st != LCA_OK) return st;
    if (P.bh == 0 || P.G == 0) return LCA_OK;
    if (out == nullptr || !aligned16(out)) return fail(LCA_ERR_INVALID_ARGUMENT, "out must be non-NULL and 16-byte aligned");
    if (lse != nullptr && (reinterpret_cast<uintptr_t>(lse) & 3u))
        return fail(LCA_ERR_INVALID_ARGUMENT, "lse must be 4-byte aligned");
    int dev = 0;
    int* err_word = nullptr;
    if ((st = check_device(&dev, &err_word)) != LCA_OK) return st;
    const Layout L = make_layout(P);
    if ((st = check_workspace(L, workspace, workspace_bytes)) != LCA_OK) return st;
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    lca::CombineParams cp;
    memset(&cp, 0, sizeof(cp));
    cp.bh = (int)P.bh;
    cp.num_global = (int)P.G;
    cp.n_parts = (int)P.world;
    cp.split_tiles = 0;  // every shard's partial is present
    cp.part_stride_o = L.rowpart_bytes / 4;
    cp.part_stride_lse = L.rowpart_bytes / 4;
    cp.part_o = reinterpret_cast<const float*>(ws + L.off_rowpart_all);
    cp.part_lse = cp.part_o + (size_t)P.bh * P.G * P.d;
    cp.gidx = reinterpret_cast<const int*>(ws + L.off_gidx);
    cp.o = out;
    cp.heads = (int)P.heads;
    cp.o_b = P.s_b();
    cp.o_h = P.s_h();
    cp.o_n = P.s_n();
    cp.lse = lse;
    cp.n_rows = (int)P.n;
    cp.row_off = (int)P.q_off;
    cudaError_t e = lca::launch_combine((int)P.d, cp, static_cast<cudaStream_t>(stream_ptr));
    if (e != cudaSuccess) return fail_cuda(e, "shard combine launch");
    return LCA_OK;
}

// ------------------------------------------------------------------ peer-memory exchange

int lca_peer_alloc(size_t bytes, void** dev_ptr, void* ipc_handle) {
    if (dev_ptr == nullptr || ipc_handle == nullptr) return fail(LCA_ERR_INVALID_ARGUMENT, "NULL output");
    *dev_ptr = nullptr;
    void* p = nullptr;
    cudaError_t e = cudaMalloc(&p, bytes > 0 ? bytes : 1);
    if (e != cudaSuccess) return fail_cuda(e, "cudaMalloc(peer workspace)");
    e = cudaMemset(p, 0, bytes > 0 ? bytes : 1);
    if (e == cudaSuccess) e = cudaIpcGetMemHandle(static_cast<cudaIpcMemHandle_t*>(ipc_handle), p);
    if (e != cudaSuccess) {
        cudaFree(p);
        return fail_cuda(e, "peer workspace setup");
    }
    *dev_ptr = p;
    return LCA_OK;
}

int lca_peer_open(const void* ipc_handle, void** dev_ptr) {
    if (dev_ptr == nullptr || ipc_handle == nullptr) return fail(LCA_ERR_INVALID_ARGUMENT, "NULL argument");
    cudaIpcMemHandle_t h;
    memcpy(&h, ipc_handle, sizeof(h));
    cudaError_t e = cudaIpcOpenMemHandle(dev_ptr, h, cudaIpcMemLazyEnablePeerAccess);
    if (e != cudaSuccess) return fail_cuda(e, "cudaIpcOpenMemHandle");
    return LCA_OK;
}

int lca_peer_close(void* dev_ptr) {
    cudaError_t e = cudaIpcCloseMemHandle(dev_ptr);
    return e == cudaSuccess ? LCA_OK : fail_cuda(e, "cudaIpcCloseMemHandle");
}

int lca_peer_free(void* dev_ptr) {
    cudaError_t e = cudaFree(dev_ptr);
    return e == cudaSuccess ? LCA_OK : fail_cuda(e, "cudaFree(peer workspace)");
}

}  // extern "C"

namespace {

int check_peer_args(const Problem& P, void* const* peers, size_t workspace_bytes, const Layout& L) {
    if (P.world > lca::kMaxPeers)
        return fail(LCA_ERR_UNSUPPORTED, "peer exchange supports at most %d ranks (got %lld)", lca::kMaxPeers,
                    (long long)P.world);
    if (peers == nullptr) return fail(LCA_ERR_INVALID_ARGUMENT, "peer workspace array is NULL");
    for (int64_t r = 0; r < P.world; ++r)
        if (peers[r] == nullptr || (reinterpret_cast<uintptr_t>(peers[r]) % 256) != 0)
            return fail(LCA_ERR_WORKSPACE, "peer workspace %lld is NULL or not 256-byte aligned", (long long)r);
    if (workspace_bytes < L.total)
        return fail(LCA_ERR_WORKSPACE, "workspace needs %zu bytes, got %zu", L.total, workspace_bytes);
    return LCA_OK;
}

uint8_t* at(void* const* peers, int64_t r, size_t off) { return static_cast<uint8_t*>(peers[r]) + off; }

}  // namespace

extern "C" {

int lca_swa_shard_exchange_peer(const lca_shard_desc* desc, const int64_t* global_tokens, int64_t num_global_tokens,
                                void* const* peer_workspaces, size_t workspace_bytes, void* stream_ptr) {
    g_last_error.clear();
    Problem P;
    int st = parse_shard(P, desc, global_tokens, num_global_tokens);
    if (st != LCA_OK) return st;
    int dev = 0;
    int* err_word = nullptr;
    if ((st = check_device(&dev, &err_word)) != LCA_OK) return st;
    const Layout L = make_layout(P);
    if ((st = check_peer_args(P, peer_workspaces, workspace_bytes, L)) != LCA_OK) return st;
    const int64_t rank = desc->rank;
    lca::PeerPutParams pp;
    memset(&pp, 0, sizeof(pp));
    pp.world = (int)P.world;
    // this rank's run of compact global rows, to every other rank
    int64_t g_lo = 0, g_hi = 0;
    for (size_t i = 0; i < P.gl.size(); ++i) {
        if (P.gl[i] < P.q_off) g_lo = (int64_t)i + 1;
        if (P.gl[i] < P.q_off + P.n) g_hi = (int64_t)i + 1;
    }
    if (g_hi > g_lo) {
        const size_t off = L.off_globals + (size_t)g_lo * L.grow_bytes;
        for (int64_t r = 0; r < P.world; ++r) {
            if (r == rank) continue;
            pp.src[pp.n_jobs] = at(peer_workspaces, rank, off);
            pp.dst[pp.n_jobs] = at(peer_workspaces, r, off);
            pp.bytes[pp.n_jobs] = (unsigned long long)(g_hi - g_lo) * L.grow_bytes;
            ++pp.n_jobs;
        }
    }
    // halo blocks: side 0 (first rows) to rank - 1's side 1, side 1 (last rows) to rank + 1's side 0
    if (L.halo_block > 0) {
        if (rank > 0) {
            pp.src[pp.n_jobs] = at(peer_workspaces, rank, L.off_send);
            pp.dst[pp.n_jobs] = at(peer_workspaces, rank - 1, L.off_recv + L.halo_block);
            pp.bytes[pp.n_jobs++] = L.halo_block;
        }
        if (rank < P.world - 1) {
            pp.src[pp.n_jobs] = at(peer_workspaces, rank, L.off_send + L.halo_block);
            pp.dst[pp.n_jobs] = at(peer_workspaces, rank + 1, L.off_recv);
            pp.bytes[pp.n_jobs++] = L.halo_block;
        }
    }
    for (int64_t r = 0; r < P.world; ++r) {
        if (r == rank) continue;
        pp.signal[r] = reinterpret_cast<unsigned int*>(at(peer_workspaces, r, L.off_sig) +
                                                       offsetof(lca::PeerSignals, prep) + rank * sizeof(unsigned int));
        pp.wait[r] = reinterpret_cast<unsigned int*>(at(peer_workspaces, rank, L.off_sig) +
                                                     offsetof(lca::PeerSignals, prep) + r * sizeof(unsigned int));
    }
    pp.epoch = reinterpret_cast<const unsigned int*>(at(peer_workspaces, rank, L.off_sig) +
                                                     offsetof(lca::PeerSignals, epoch));
    pp.err = err_word;
    pp.timeout_ns = wait_timeout_ns();
    cudaError_t e = lca::launch_peer_put(pp, lca::kPeerPrepBlocks, static_cast<cudaStream_t>(stream_ptr));
    if (e != cudaSuccess) return fail_cuda(e, "peer exchange launch");
    return LCA_OK;
}

int lca_swa_shard_finish_peer(const lca_shard_desc* desc, float* out, float* lse, const int64_t* global_tokens,
                              int64_t num_global_tokens, void* const* peer_workspaces, size_t workspace_bytes,
                              void* stream_ptr) {
    g_last_error.clear();
    Problem P;
    int st = parse_shard(P, desc, global_tokens, num_global_tokens);
    if (st != LCA_OK) return st;
    if (P.G > 0 && (out == nullptr || !aligned16(out)))
        return fail(LCA_ERR_INVALID_ARGUMENT, "out must be non-NULL and 16-byte aligned");
    int dev = 0;
    int* err_word = nullptr;
    if ((st = check_device(&dev, &err_word)) != LCA_OK) return st;
    const Layout L = make_layout(P);
    if ((st = check_peer_args(P, peer_workspaces, workspace_bytes, L)) != LCA_OK) return st;
    const int64_t rank = desc->rank;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
    uint8_t* own_sig = at(peer_workspaces, rank, L.off_sig);
    // 1. this rank's row partial into slot `rank` of every rank's gathered region (the
    //    buffer of the step's parity), then signal and wait: also the end-of-step barrier
    //    that keeps any rank from overwriting buffers another rank still reads
    lca::PeerPutParams pp;
    memset(&pp, 0, sizeof(pp));
    pp.world = (int)P.world;
    if (L.rowpart_bytes > 0) {
        for (int64_t r = 0; r < P.world; ++r) {
            pp.src[pp.n_jobs] = at(peer_workspaces, rank, L.off_rowpart);
            pp.dst[pp.n_jobs] = at(peer_workspaces, r, L.off_rowpart_all + (size_t)rank * L.rowpart_bytes);
            pp.bytes[pp.n_jobs] = L.rowpart_bytes;
            pp.parity_bytes[pp.n_jobs] = (unsigned long long)P.world * L.rowpart_bytes;
            ++pp.n_jobs;
        }
    }
    for (int64_t r = 0; r < P.world; ++r) {
        if (r == rank) continue;
        pp.signal[r] = reinterpret_cast<unsigned int*>(at(peer_workspaces, r, L.off_sig) +
                                                       offsetof(lca::PeerSignals, fin) + rank * sizeof(unsigned int));
        pp.wait[r] = reinterpret_cast<unsigned int*>(own_sig + offsetof(lca::PeerSignals, fin) +
                                                     r * sizeof(unsigned int));
    }
    pp.epoch = reinterpret_cast<const unsigned int*>(own_sig + offsetof(lca::PeerSignals, epoch));
    pp.err = err_word;
    pp.timeout_ns = wait_timeout_ns();
    cudaError_t e = lca::launch_peer_put(pp, lca::kPeerCopyBlocks, stream);
    if (e != cudaSuccess) return fail_cuda(e, "peer row-partial launch");
    // 2. merge over the shards' partials into the global rows this shard owns; its last
    //    block advances the epoch
    lca::CombineParams cp;
    memset(&cp, 0, sizeof(cp));
    cp.bh = (int)P.bh;
    cp.num_global = (int)P.G;
    cp.n_parts = (int)P.world;
    cp.split_tiles = 0;
    cp.part_stride_o = L.rowpart_bytes / 4;
    cp.part_stride_lse = L.rowpart_bytes / 4;
    cp.part_o = reinterpret_cast<const float*>(at(peer_workspaces, rank, L.off_rowpart_all));
    cp.part_lse = cp.part_o + (size_t)P.bh * P.G * P.d;
    cp.gidx = reinterpret_cast<const int*>(at(peer_workspaces, rank, L.off_gidx));
    cp.o = out;
    cp.heads = (int)P.heads;
    cp.o_b = P.s_b();
    cp.o_h = P.s_h();
    cp.o_n = P.s_n();
    cp.lse = lse;
    cp.n_rows = (int)P.n;
    cp.row_off = (int)P.q_off;
    cp.epoch = reinterpret_cast<unsigned int*>(own_sig + offsetof(lca::PeerSignals, epoch));
    cp.ticket = reinterpret_cast<unsigned int*>(own_sig + offsetof(lca::PeerSignals, ticket));
    cp.parity_floats = (size_t)P.world * L.rowpart_bytes / 4;
    e = lca::launch_combine((int)P.d, cp, stream);
    if (e != cudaSuccess) return fail_cuda(e, "peer merge launch");
    return LCA_OK;
}

int lca_set_timing_events(void* before_main, void* after_main) {
    g_ev_before_main = static_cast<cudaEvent_t>(before_main);
    g_ev_after_main = static_cast<cudaEvent_t>(after_main);
    return LCA_OK;
}

int lca_device_error(int* code) {
    if (code == nullptr) return fail(LCA_ERR_INVALID_ARGUMENT, "code is NULL");
    int dev = 0;
    int* err_word = nullptr;
    int st = check_device(&dev, &err_word);
    if (st != LCA_OK) return st;
    cudaError_t e = cudaDeviceSynchronize();
    if (e != cudaSuccess) return fail_cuda(e, "cudaDeviceSynchronize");
    int val = 0;
    e = cudaMemcpy(&val, err_word, sizeof(int), cudaMemcpyDeviceToHost);
    if (e != cudaSuccess) return fail_cuda(e, "read error word");
    const int zero = 0;
    e = cudaMemcpy(err_word, &zero, sizeof(int), cudaMemcpyHostToDevice);
    if (e != cudaSuccess) return fail_cuda(e, "clear error word");
    *code = val;
    return LCA_OK;
}

}  // extern "C"

// ------------------------------------------------------------------ backward pass

namespace {

// Workspace of the backward: the 16-bit dO, per-row stats, the global index list, the
// compact global rows ([G][4 (q, k, v, dO16)][bh][d]) with their stats, and the split
// partials of the global-row and global-key units.
constexpr int kBwdInnerRows = 64;  // rows of an inner tile of the backward kernels

struct BwdLayout {
    int n_tiles = 0, g_tiles = 0, gi_tiles = 0, split_tiles = 0, n_splits = 0;
    size_t off_dout16 = 0, off_lse2 = 0, off_dvec = 0, off_gidx = 0, off_bitmap = 0, off_compact = 0, off_lse2g = 0,
           off_dg = 0;
    int bitmap_words = 0;
    size_t off_pq = 0, off_pk = 0, off_pv = 0, total = 0;
};

BwdLayout make_bwd_layout(const Problem& P) {
    BwdLayout B;
    const size_t bh = (size_t)P.bh, n = (size_t)P.n, d = (size_t)P.d, G = (size_t)P.G;
    B.n_tiles = (int)((P.n + lca::kTileRows - 1) / lca::kTileRows);
    if (G > 0) {
        B.g_tiles = (int)((P.G + lca::kTileRows - 1) / lca::kTileRows);
        B.gi_tiles = (int)((P.G + kBwdInnerRows - 1) / kBwdInnerRows);
        // a split is about twice a band unit's inner tiles
        const int64_t band_tiles = (2 * P.window + lca::kTileRows + 2 * kBwdInnerRows - 1) / kBwdInnerRows + B.gi_tiles;
        B.split_tiles = (int)std::max<int64_t>(16, std::min<int64_t>(128, 2 * band_tiles));
        const int64_t inner_tiles = (P.n + kBwdInnerRows - 1) / kBwdInnerRows;
        B.n_splits = (int)((inner_tiles + B.split_tiles - 1) / B.split_tiles);
    }
    size_t off = 0;
    auto take = [&](size_t& at, size_t bytes) {
        at = off;
        off = align_up(off + bytes, kAlign);
    };
    take(B.off_dout16, bh * n * d * 2);
    take(B.off_lse2, bh * n * 4);
    take(B.off_dvec, bh * n * 4);
    if (G > 0) {
        take(B.off_gidx, G * 4);
        B.bitmap_words = (int)((n + 31) / 32 + 3);
        take(B.off_bitmap, (size_t)B.bitmap_words * 4);
        take(B.off_compact, G * 4 * bh * d * 2);
        take(B.off_lse2g, bh * G * 4);
        take(B.off_dg, bh * G * 4);
        const size_t part = (size_t)B.n_splits * bh * G * d * 4;
        take(B.off_pq, part);
        take(B.off_pk, part);
        take(B.off_pv, part);
    }
    B.total = off;
    return B;
}

}  // namespace

extern "C" {

int lca_swa_backward_workspace_size(int64_t batch, int64_t heads, int64_t seq_len, int64_t head_dim,
                                    int64_t window_size, int64_t num_unique_global, int dtype, size_t* out_bytes) {
    g_last_error.clear();
    if (out_bytes == nullptr) return fail(LCA_ERR_INVALID_ARGUMENT, "out_bytes is NULL");
    if (batch < 0 || heads < 0 || seq_len < 0 || num_unique_global < 0)
        return fail(LCA_ERR_INVALID_ARGUMENT, "negative size");
    int st = check_dtype_dim(dtype, head_dim);
    if (st != LCA_OK) return st;
    if (window_size < 0) return fail(LCA_ERR_INVALID_ARGUMENT, "window_size must be >= 0");
    Problem P;
    P.bh = batch * heads;
    P.n_total = P.n = seq_len;
    P.d = head_dim;
    P.window = std::min(window_size, seq_len);
    P.G = std::min(num_unique_global, seq_len);
    P.dtype = dtype;
    *out_bytes = make_bwd_layout(P).total;
    return LCA_OK;
}

int lca_swa_backward(const void* q, const void* k, const void* v, const float* o, const float* lse,
                     const float* dout, float* dq, float* dk, float* dv, int dtype, int64_t batch, int64_t heads,
                     int64_t seq_len, int64_t head_dim, int64_t window_size, float scale,
                     const int64_t* global_tokens, int64_t num_global_tokens, void* workspace,
                     size_t workspace_bytes, void* stream_ptr) {
    g_last_error.clear();
    Problem P;
    int st = parse_common(P, dtype, batch, heads, seq_len, head_dim, window_size, scale, global_tokens,
                          num_global_tokens);
    if (st != LCA_OK) return st;
    if (P.bh == 0 || P.n == 0) return LCA_OK;
    const void* ptrs[9] = {q, k, v, o, lse, dout, dq, dk, dv};
    for (const void* x : ptrs)
        if (x == nullptr) return fail(LCA_ERR_INVALID_ARGUMENT, "q, k, v, o, lse, dout, dq, dk and dv must be non-NULL");
    for (int i = 0; i < 9; ++i)
        if (i != 4 && !aligned16(ptrs[i]))
            return fail(LCA_ERR_INVALID_ARGUMENT, "q, k, v, o, dout, dq, dk and dv must be 16-byte aligned");
    if (reinterpret_cast<uintptr_t>(lse) & 3u) return fail(LCA_ERR_INVALID_ARGUMENT, "lse must be 4-byte aligned");
    if (P.bh * (int64_t)((P.n + lca::kTileRows - 1) / lca::kTileRows) > INT_MAX / 2)
        return fail(LCA_ERR_UNSUPPORTED, "problem too large for the backward");
    int dev = 0;
    int* err_word = nullptr;
    if ((st = check_device(&dev, &err_word)) != LCA_OK) return st;
    const BwdLayout B = make_bwd_layout(P);
    if (workspace_bytes < B.total)
        return fail(LCA_ERR_WORKSPACE, "backward workspace needs %zu bytes, got %zu", B.total, workspace_bytes);
    if (B.total > 0 && (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) % 256) != 0))
        return fail(LCA_ERR_WORKSPACE, "workspace must be non-NULL and 256-byte aligned");
    cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    const bool bf16 = P.dtype == LCA_DTYPE_BF16;
    const int d = (int)P.d;
    const int G = (int)P.G;
    int* gidx = G > 0 ? reinterpret_cast<int*>(ws + B.off_gidx) : nullptr;
    cudaError_t e;

    // 1. the sorted global indices
    for (int first = 0; first < G; first += lca::kBwdIndexChunk) {
        static thread_local lca::BwdIndexParams ip;
        ip.dst = gidx + first;
        ip.bitmap = reinterpret_cast<uint32_t*>(ws + B.off_bitmap);
        ip.bitmap_words = B.bitmap_words;
        ip.clear_bitmap = first == 0 ? 1 : 0;
        ip.count = std::min(lca::kBwdIndexChunk, G - first);
        for (int i = 0; i < ip.count; ++i) ip.idx[i] = P.gl[(size_t)first + i];
        if ((e = lca::launch_bwd_indices(ip, stream)) != cudaSuccess) return fail_cuda(e, "backward index launch");
    }
    // 2. per-row preparation
    lca::BwdPrepParams pp;
    memset(&pp, 0, sizeof(pp));
    pp.q = q;
    pp.k = k;
    pp.v = v;
    pp.o = o;
    pp.dout = dout;
    pp.lse = lse;
    pp.dout16 = ws + B.off_dout16;
    pp.lse2 = reinterpret_cast<float*>(ws + B.off_lse2);
    pp.dvec = reinterpret_cast<float*>(ws + B.off_dvec);
    if (G > 0) {
        pp.compact = ws + B.off_compact;
        pp.lse2g = reinterpret_cast<float*>(ws + B.off_lse2g);
        pp.dg = reinterpret_cast<float*>(ws + B.off_dg);
    }
    pp.gidx = gidx;
    pp.gbitmap = G > 0 ? reinterpret_cast<const uint32_t*>(ws + B.off_bitmap) : nullptr;
    pp.num_global = G;
    pp.n = (int)P.n;
    pp.bh = (int)P.bh;
    pp.bf16 = bf16 ? 1 : 0;
    if ((e = lca::launch_bwd_prep(d, pp, stream)) != cudaSuccess) return fail_cuda(e, "backward prep launch");

    // 3. tensor maps: the inputs, the 16-bit dO and the compact planes
    const CUtensorMapDataType dt = bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    // [0] outer tiles (128-row boxes), [1] inner tiles (64-row boxes)
    CUtensorMap mq[2], mk[2], mv[2], mdo[2], mqg[2], mkg[2], mvg[2], mdog[2];
    const uint64_t rows = (uint64_t)P.n, planes = (uint64_t)P.bh;
    const void* dout16 = ws + B.off_dout16;
    for (int i = 0; i < 2; ++i) {
        const uint32_t br = i == 0 ? lca::kTileRows : kBwdInnerRows;
        const CUtensorMapSwizzle sw = CU_TENSOR_MAP_SWIZZLE_128B;
        if ((st = encode_3d(&mq[i], dt, 2, q, d, rows, planes, 64, "q", sw, br)) != LCA_OK) return st;
        if ((st = encode_3d(&mk[i], dt, 2, k, d, rows, planes, 64, "k", sw, br)) != LCA_OK) return st;
        if ((st = encode_3d(&mv[i], dt, 2, v, d, rows, planes, 64, "v", sw, br)) != LCA_OK) return st;
        if ((st = encode_3d(&mdo[i], dt, 2, dout16, d, rows, planes, 64, "dout16", sw, br)) != LCA_OK) return st;
        if (G > 0) {
            const uint8_t* cb = ws + B.off_compact;
            const size_t pb = (size_t)P.bh * d * 2;
            if ((st = encode_compact(&mqg[i], dt, cb, d, planes, G, "q global rows", 4, br)) != LCA_OK) return st;
            if ((st = encode_compact(&mkg[i], dt, cb + pb, d, planes, G, "k global rows", 4, br)) != LCA_OK) return st;
            if ((st = encode_compact(&mvg[i], dt, cb + 2 * pb, d, planes, G, "v global rows", 4, br)) != LCA_OK)
                return st;
            if ((st = encode_compact(&mdog[i], dt, cb + 3 * pb, d, planes, G, "dout16 global rows", 4, br)) != LCA_OK)
                return st;
        } else {  // never loaded without global tokens
            mqg[i] = mq[i];
            mkg[i] = mk[i];
            mvg[i] = mv[i];
            mdog[i] = mdo[i];
        }
    }

    // 4. the dQ kernel and the dK / dV kernel
    lca::BwdParams bp;
    memset(&bp, 0, sizeof(bp));
    bp.n = (int)P.n;
    bp.bh = (int)P.bh;
    bp.window = (int)P.window;
    bp.num_global = G;
    bp.g_tiles = B.g_tiles;
    bp.gi_tiles = B.gi_tiles;
    bp.n_tiles = B.n_tiles;
    bp.split_tiles = B.split_tiles;
    bp.n_splits = B.n_splits;
    bp.n_band_units = (int)(P.bh * B.n_tiles);
    const long long units = (long long)bp.n_band_units + (long long)P.bh * B.g_tiles * B.n_splits;
    if (units > INT_MAX) return fail(LCA_ERR_UNSUPPORTED, "problem too large (%lld backward units)", units);
    bp.n_units = (int)units;
    bp.grid = g_dev_sms[dev] > 0 ? g_dev_sms[dev] : 148;
    bp.scale = scale;
    bp.scale_log2 = scale * 1.4426950408889634f;
    bp.gidx = gidx;
    bp.gbitmap = G > 0 ? reinterpret_cast<const uint32_t*>(ws + B.off_bitmap) : nullptr;
    bp.lse2 = pp.lse2;
    bp.dvec = pp.dvec;
    bp.lse2g = pp.lse2g;
    bp.dg = pp.dg;
    bp.err = err_word;
    bp.timeout_ns = wait_timeout_ns();
    float* pq = G > 0 ? reinterpret_cast<float*>(ws + B.off_pq) : nullptr;
    float* pk = G > 0 ? reinterpret_cast<float*>(ws + B.off_pk) : nullptr;
    float* pv = G > 0 ? reinterpret_cast<float*>(ws + B.off_pv) : nullptr;

    lca::BwdMaps mqk{mq[0], mdo[0], mk[1], mv[1], mqg[0], mdog[0], mkg[1], mvg[1]};  // outer (Q, dO16), inner (K, V)
    lca::BwdParams bq = bp;
    bq.out_a = dq;
    bq.part_a = pq;
    if ((e = lca::launch_bwd_main(d, bf16, false, mqk, bq, stream)) != cudaSuccess)
        return fail_cuda(e, "backward dQ kernel launch");
    lca::BwdMaps mkv{mk[0], mv[0], mq[1], mdo[1], mkg[0], mvg[0], mqg[1], mdog[1]};  // outer (K, V), inner (Q, dO16)
    lca::BwdParams bk = bp;
    bk.out_a = dv;
    bk.out_b = dk;
    bk.part_a = pv;
    bk.part_b = pk;
    if ((e = lca::launch_bwd_main(d, bf16, true, mkv, bk, stream)) != cudaSuccess)
        return fail_cuda(e, "backward dK/dV kernel launch");

    // 5. the global tokens' rows
    if (G > 0) {
        lca::BwdReduceParams rp;
        memset(&rp, 0, sizeof(rp));
        rp.part_q = pq;
        rp.part_k = pk;
        rp.part_v = pv;
        rp.dq = dq;
        rp.dk = dk;
        rp.dv = dv;
        rp.gidx = gidx;
        rp.splits_q = rp.splits_k = B.n_splits;
        rp.num_global = G;
        rp.n = (int)P.n;
        rp.bh = (int)P.bh;
        if ((e = lca::launch_bwd_reduce(d, rp, stream)) != cudaSuccess) return fail_cuda(e, "backward reduce launch");
    }
    return LCA_OK;
}

#ifdef LCA_TRACE
// Trace builds only (not in the public header): copy the main kernel's event trace out.
LCA_API int lca_trace_read(void* host, size_t bytes) {
    if (host == nullptr) return fail(LCA_ERR_INVALID_ARGUMENT, "host is NULL");
    cudaError_t e = cudaDeviceSynchronize();
    if (e == cudaSuccess) e = lca::trace_read(host, bytes);
    if (e != cudaSuccess) return fail_cuda(e, "trace read");
    return LCA_OK;
}
#endif

}  // extern "C"
