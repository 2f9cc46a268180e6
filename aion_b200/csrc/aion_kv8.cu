// Host side of the 8-bit paged K/V cache (aion_kv8_* of include/aion.h):
// checks of the arguments, launches.  Nothing here waits for the device but
// aion_kv8_create and aion_kv8_status.
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>
#include <mutex>
#include <utility>

#include "kv8.h"
#include "kv8.cuh"
#include "kv8_attention.cuh"
#include "kv8_prompt.cuh"

using namespace aion;

// A failed call leaves its error behind for cudaGetLastError, too: taken here,
// or the next launch that is checked would seem to have failed.
#define KV_CUDA(call)                                                                                       \
    do {                                                                                                    \
        cudaError_t e_ = (call);                                                                            \
        if (e_ != cudaSuccess) {                                                                            \
            (void)cudaGetLastError();                                                                       \
            aion_thread_error("%s: CUDA error %s (%s)", what, cudaGetErrorName(e_), cudaGetErrorString(e_)); \
            return e_ == cudaErrorMemoryAllocation ? AION_ERR_OOM : AION_ERR_CUDA;                          \
        }                                                                                                   \
    } while (0)

#define KV_ARG(cond, ...)                 \
    do {                                  \
        if (!(cond)) {                    \
            aion_thread_error(__VA_ARGS__); \
            return AION_ERR_ARG;          \
        }                                 \
    } while (0)

// Makes `dev` current for the call and the caller's device current again after it.
struct DeviceGuard {
    int before = -1;
    cudaError_t err;
    explicit DeviceGuard(int dev) {
        err = cudaGetDevice(&before);
        if (err == cudaSuccess && before != dev) err = cudaSetDevice(dev);
        else if (err == cudaSuccess) before = -1;
    }
    ~DeviceGuard() {
        if (before >= 0) cudaSetDevice(before);
    }
};

static aion_status check_shape(const aion_kv8* kv, const char* what) {
    KV_ARG(kv, "%s: null cache", what);
    const bool page_ok = kv->page_tokens == 16 || kv->page_tokens == 32 || kv->page_tokens == 64 || kv->page_tokens == 128;
    if (!page_ok || kv->head_size < 16 || kv->head_size > kKvMaxHead || kv->head_size % 16) {
        aion_thread_error("%s: page_tokens %d must be 16, 32, 64 or 128 and head_size %d a multiple of 16 up to %d", what,
                          kv->page_tokens, kv->head_size, kKvMaxHead);
        return AION_ERR_SHAPE;
    }
    if (kv->n_layers < 1 || kv->n_pages < 1 || kv->n_kv_heads < 1 || kv->n_kv_heads > 65535 || kv->max_seqs < 1 ||
        kv->max_seqs > kKvMaxSeqs || kv->max_pages < 1 || kv->n_pages > (1 << 24) || kv->n_layers > 65535 ||
        (int64_t)kv->max_pages * kv->page_tokens > (1 << 30)) {
        aion_thread_error("%s: %d layers, %d pages, %d K/V heads, %d slots (at most %d) of %d pages are out of range", what,
                          kv->n_layers, kv->n_pages, kv->n_kv_heads, kv->max_seqs, kKvMaxSeqs, kv->max_pages);
        return AION_ERR_SHAPE;
    }
    // Each count is in range, but sizes in bytes and offsets are products of them in 64 bits.
    if ((double)kv->n_layers * kv->n_pages * kv->n_kv_heads * kv->page_tokens * kv->head_size > 1152921504606846976.0) {   // 2^60
        aion_thread_error("%s: %d layers of %d pages of %d x %d x %d values pass 2^60 bytes", what, kv->n_layers, kv->n_pages,
                          kv->n_kv_heads, kv->page_tokens, kv->head_size);
        return AION_ERR_SHAPE;
    }
    return AION_OK;
}

static aion_status check_cache(const aion_kv8* kv, const char* what) {
    const aion_status s = check_shape(kv, what);
    if (s != AION_OK) return s;
    KV_ARG(kv->k && kv->v && kv->k_scale && kv->v_scale && kv->tables && kv->lens && kv->refs && kv->work,
           "%s: the cache has a null pointer", what);
    KV_ARG((((uintptr_t)kv->k | (uintptr_t)kv->v) & 15) == 0, "%s: k and v must be 16-byte aligned", what);
    KV_ARG((((uintptr_t)kv->k_scale | (uintptr_t)kv->v_scale | (uintptr_t)kv->tables | (uintptr_t)kv->lens |
             (uintptr_t)kv->refs | (uintptr_t)kv->work) & 3) == 0,
           "%s: scales, tables, lens, refs and work must be 4-byte aligned", what);
    return AION_OK;
}

static KvView view_of(const aion_kv8* kv) {
    KvView c;
    c.k = kv->k;
    c.v = kv->v;
    c.k_scale = kv->k_scale;
    c.v_scale = kv->v_scale;
    c.tables = kv->tables;
    c.lens = kv->lens;
    c.refs = kv->refs;
    c.work = kv->work;
    c.n_layers = kv->n_layers;
    c.n_pages = kv->n_pages;
    c.nkv = kv->n_kv_heads;
    c.page = kv->page_tokens;
    c.page_log = kv->page_tokens == 16 ? 4 : kv->page_tokens == 32 ? 5 : kv->page_tokens == 64 ? 6 : 7;
    c.hd = kv->head_size;
    c.max_seqs = kv->max_seqs;
    c.max_pages = kv->max_pages;
    return c;
}

static int sm_count(int dev) {
    static int sms[64] = {};   // written with one value only: a race is harmless
    if (dev < 0 || dev >= 64) return 148;
    if (!sms[dev]) {
        int v = 0;
        if (cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) {
            (void)cudaGetLastError();
            return 148;
        }
        sms[dev] = v;
    }
    return sms[dev];
}

template <typename... KArgs, typename... Args>
static cudaError_t launch_pdl(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st,
                              Args&&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}

// ---------------------------------------------------------------------------
// The cache
// ---------------------------------------------------------------------------
extern "C" AION_API aion_status aion_kv8_create(const aion_kv8* shape, aion_kv8* out) {
    const char* what = "aion_kv8_create";
    KV_ARG(out, "%s: null result", what);
    const aion_status s = check_shape(shape, what);
    if (s != AION_OK) return s;
    aion_kv8 kv = *shape;
    DeviceGuard dev(kv.device);
    KV_CUDA(dev.err);
    auto up = [](int64_t b) { return (b + 255) & ~(int64_t)255; };
    const int64_t pool = up((int64_t)kv.n_layers * kv.n_pages * kv.n_kv_heads * kv.page_tokens * kv.head_size);
    const int64_t sc = up((int64_t)kv.n_layers * kv.n_pages * kv.n_kv_heads * 4);
    const int64_t tab = up((int64_t)kv.max_seqs * kv.max_pages * 4), len = up((int64_t)kv.max_seqs * 4);
    const int64_t ref = up((int64_t)kv.n_pages * 4), work = up((4 + 3 * (int64_t)kv.n_pages) * 4);
    char* p = nullptr;
    const int64_t total = 2 * pool + 2 * sc + tab + len + ref + work;
    KV_CUDA(cudaMalloc(&p, total));
    kv.k = (int8_t*)p;
    kv.v = (int8_t*)(p + pool);
    kv.k_scale = (float*)(p + 2 * pool);
    kv.v_scale = (float*)(p + 2 * pool + sc);
    kv.tables = (int32_t*)(p + 2 * pool + 2 * sc);
    kv.lens = (int32_t*)(p + 2 * pool + 2 * sc + tab);
    kv.refs = (int32_t*)(p + 2 * pool + 2 * sc + tab + len);
    kv.work = (int32_t*)(p + 2 * pool + 2 * sc + tab + len + ref);
    cudaError_t e = cudaMemset(p, 0, total);
    if (e == cudaSuccess) e = cudaMemset(kv.tables, 0xFF, (int64_t)kv.max_seqs * kv.max_pages * 4);
    if (e == cudaSuccess) e = cudaDeviceSynchronize();
    if (e != cudaSuccess) {
        cudaFree(p);
        KV_CUDA(e);
    }
    *out = kv;
    return AION_OK;
}

extern "C" AION_API aion_status aion_kv8_destroy(aion_kv8* kv) {
    const char* what = "aion_kv8_destroy";
    if (!kv || !kv->k) return AION_OK;
    DeviceGuard dev(kv->device);
    KV_CUDA(dev.err);
    KV_CUDA(cudaFree(kv->k));
    *kv = aion_kv8();
    return AION_OK;
}

extern "C" AION_API aion_status aion_kv8_reset(const aion_kv8* kv, void* stream) {
    const char* what = "aion_kv8_reset";
    const aion_status s = check_cache(kv, what);
    if (s != AION_OK) return s;
    DeviceGuard dev(kv->device);
    KV_CUDA(dev.err);
    const int64_t n = std::max<int64_t>((int64_t)kv->max_seqs * kv->max_pages, kv->n_pages);
    k_kv_reset<<<(int)std::min<int64_t>((n + 255) / 256, 1184), 256, 0, (cudaStream_t)stream>>>(view_of(kv));
    KV_CUDA(cudaGetLastError());
    return AION_OK;
}

static aion_status check_list(const aion_kv8* kv, const void* a, const void* b, int n, const char* what) {
    const aion_status s = check_cache(kv, what);
    if (s != AION_OK) return s;
    KV_ARG(n >= 0 && n <= kKvMaxList, "%s: %d entries (at most %d)", what, n, kKvMaxList);
    KV_ARG(n == 0 || (a && b), "%s: null list", what);
    return AION_OK;
}

// The page copies of the lists that the kernel before has made.
static cudaError_t launch_move(const aion_kv8* kv, int tables, cudaStream_t st) {
    // As many blocks as an SM takes, and no more than a call could use: 16 sequences of 7B leave, compacted in 310 us
    // with 6 an SM, 340 with 4, 336 with 8 of fewer registers.
    const int64_t units = ((int64_t)kv->n_kv_heads * kv->page_tokens * kv->head_size + kKvCopyUnit - 1) / kKvCopyUnit;
    const int64_t most = units * kv->n_layers * 2 * kv->n_pages;
    const int grid = (int)std::min<int64_t>(most, (int64_t)sm_count(kv->device) * 6);
    return launch_pdl(k_kv_move, dim3(grid), dim3(kKvCopyThreads), 0, st, view_of(kv), tables);
}

extern "C" AION_API aion_status aion_kv8_grow(const aion_kv8* kv, const int32_t* seqs, const int32_t* n_new, int32_t n,
                                              int32_t* pos0, void* stream) {
    const char* what = "aion_kv8_grow";
    const aion_status s = check_list(kv, seqs, n_new, n, what);
    if (s != AION_OK) return s;
    KV_ARG(n == 0 || pos0, "%s: null pos0", what);
    if (n == 0) return AION_OK;
    DeviceGuard dev(kv->device);
    KV_CUDA(dev.err);
    k_kv_grow<<<1, 1024, 0, (cudaStream_t)stream>>>(view_of(kv), seqs, n_new, n, pos0);
    KV_CUDA(cudaGetLastError());
    KV_CUDA(launch_move(kv, 0, (cudaStream_t)stream));
    return AION_OK;
}

extern "C" AION_API aion_status aion_kv8_fork(const aion_kv8* kv, const int32_t* src, const int32_t* dst,
                                              const int32_t* keep, int32_t n, void* stream) {
    const char* what = "aion_kv8_fork";
    const aion_status s = check_list(kv, src, dst, n, what);
    if (s != AION_OK) return s;
    if (n == 0) return AION_OK;
    DeviceGuard dev(kv->device);
    KV_CUDA(dev.err);
    k_kv_fork<<<n, 128, 0, (cudaStream_t)stream>>>(view_of(kv), src, dst, keep, n);
    KV_CUDA(cudaGetLastError());
    return AION_OK;
}

extern "C" AION_API aion_status aion_kv8_trim(const aion_kv8* kv, const int32_t* seqs, const int32_t* keep, int32_t n,
                                              void* stream) {
    const char* what = "aion_kv8_trim";
    const aion_status s = check_list(kv, seqs, seqs, n, what);
    if (s != AION_OK) return s;
    if (n == 0) return AION_OK;
    DeviceGuard dev(kv->device);
    KV_CUDA(dev.err);
    k_kv_trim<<<n, 128, 0, (cudaStream_t)stream>>>(view_of(kv), seqs, keep, n);
    KV_CUDA(cudaGetLastError());
    return AION_OK;
}

extern "C" AION_API aion_status aion_kv8_compact(const aion_kv8* kv, int32_t* n_used, void* stream) {
    const char* what = "aion_kv8_compact";
    const aion_status s = check_cache(kv, what);
    if (s != AION_OK) return s;
    DeviceGuard dev(kv->device);
    KV_CUDA(dev.err);
    k_kv_compact<<<1, 1024, 0, (cudaStream_t)stream>>>(view_of(kv), n_used);
    KV_CUDA(cudaGetLastError());
    KV_CUDA(launch_move(kv, 1, (cudaStream_t)stream));
    return AION_OK;
}

// ---------------------------------------------------------------------------
// Rows
// ---------------------------------------------------------------------------
static int type_bytes(int type) { return type == AION_F32 ? 4 : 2; }

static aion_status check_rows(const aion_kv8* kv, int layer, int type, const int32_t* seqs, const int32_t* pos0,
                              const int32_t* cu, int n_seq, int n_tok, const char* what) {
    const aion_status s = check_cache(kv, what);
    if (s != AION_OK) return s;
    KV_ARG(layer >= 0 && layer < kv->n_layers, "%s: layer %d out of range [0, %d)", what, layer, kv->n_layers);
    KV_ARG(type == AION_F32 || type == AION_F16 || type == AION_BF16, "%s: unknown element type %d", what, type);
    KV_ARG(n_seq >= 0 && n_seq <= kKvMaxSeqs && n_tok >= 0 && n_tok <= (1 << 24),
           "%s: %d sequences (at most %d), %d rows (at most %d)", what, n_seq, kKvMaxSeqs, n_tok, 1 << 24);
    KV_ARG(((int64_t)(n_tok >> 4) + 2 * n_seq) * kv->n_kv_heads * 2 < ((int64_t)1 << 31), "%s: %d rows of %d heads are too many",
           what, n_tok, kv->n_kv_heads);
    KV_ARG(cu || n_seq == n_tok, "%s: without cu every sequence has one row (%d sequences, %d rows)", what, n_seq, n_tok);
    KV_ARG(n_seq == 0 || (seqs && pos0), "%s: null seqs or pos0", what);
    return AION_OK;
}

// Rows of `heads` x head_size elements: the stride holds a row; whether 16
// values may be moved as 16-byte vectors is the kernels' `vec`.
static aion_status check_matrix(const void* p, int64_t stride, int64_t width, int type, int n_tok, const char* name,
                                const char* what) {
    KV_ARG(p || n_tok == 0, "%s: null %s", what, name);
    KV_ARG((uintptr_t)p % type_bytes(type) == 0, "%s: %s is not aligned to its elements", what, name);
    KV_ARG(n_tok <= 1 || (stride >= width && stride < ((int64_t)1 << 32)),
           "%s: %s's rows are %lld elements apart and %lld wide", what, name, (long long)stride, (long long)width);
    return AION_OK;
}
static bool vectors(const void* p, int64_t stride, int type) {
    return ((uintptr_t)p & 15) == 0 && (stride * type_bytes(type)) % 16 == 0;
}

template <typename T>
static cudaError_t launch_append(const KvAppendArgs& a, cudaStream_t st) {
    if (!a.r.cu) {
        const int64_t warps = (int64_t)a.r.n_seq * a.c.nkv * 2;
        k_kv_append_one<T><<<(unsigned)((warps + kKvAppendThreads / 32 - 1) / (kKvAppendThreads / 32)), kKvAppendThreads, 0, st>>>(a);
        return cudaGetLastError();
    }
    const unsigned grid = (unsigned)((int64_t)kv_places(true, a.r.n_seq, a.r.n_tok, a.c.page_log, 2) * a.c.nkv * 2);
    if (a.c.page == 16) k_kv_append<T, 4, 128><<<grid, 128, 0, st>>>(a);
    else if (a.c.page == 32) k_kv_append<T, 8, 128><<<grid, 128, 0, st>>>(a);
    else if (a.c.page == 64) k_kv_append<T, 16, 128><<<grid, 128, 0, st>>>(a);
    else k_kv_append<T, 16, 256><<<grid, 256, 0, st>>>(a);
    return cudaGetLastError();
}

template <typename T>
static cudaError_t launch_read(const KvReadArgs& a, cudaStream_t st) {
    if (!a.r.cu) {
        const int64_t warps = (int64_t)a.r.n_seq * a.c.nkv * 2;
        k_kv_read_one<T><<<(unsigned)((warps + kKvAppendThreads / 32 - 1) / (kKvAppendThreads / 32)), kKvAppendThreads, 0, st>>>(a);
    } else {
        const int64_t grid = (int64_t)kv_places(true, a.r.n_seq, a.r.n_tok, kKvReadLog, 1) * a.c.nkv * 2;
        k_kv_read<T><<<(unsigned)grid, kKvReadThreads, 0, st>>>(a);
    }
    return cudaGetLastError();
}

extern "C" AION_API aion_status aion_kv8_append(const aion_kv8* kv, int32_t layer, const void* k, const void* v,
                                                int32_t type, int64_t k_stride, int64_t v_stride, const int32_t* seqs,
                                                const int32_t* pos0, const int32_t* cu, int32_t n_seq, int32_t n_tok,
                                                void* stream) {
    const char* what = "aion_kv8_append";
    aion_status s = check_rows(kv, layer, type, seqs, pos0, cu, n_seq, n_tok, what);
    const int64_t width = s == AION_OK ? (int64_t)kv->n_kv_heads * kv->head_size : 0;
    if (s == AION_OK) s = check_matrix(k, k_stride, width, type, n_tok, "k", what);
    if (s == AION_OK) s = check_matrix(v, v_stride, width, type, n_tok, "v", what);
    if (s != AION_OK || n_tok == 0 || n_seq == 0) return s;
    DeviceGuard dev(kv->device);
    KV_CUDA(dev.err);
    KvAppendArgs a;
    a.c = view_of(kv);
    a.r = {seqs, pos0, cu, n_seq, n_tok};
    a.layer = layer;
    a.k = k;
    a.v = v;
    a.k_stride = k_stride;
    a.v_stride = v_stride;
    a.vec = vectors(k, k_stride, type) && vectors(v, v_stride, type);
    KV_CUDA(type == AION_F32 ? launch_append<float>(a, (cudaStream_t)stream)
            : type == AION_F16 ? launch_append<__half>(a, (cudaStream_t)stream)
                               : launch_append<__nv_bfloat16>(a, (cudaStream_t)stream));
    return AION_OK;
}

extern "C" AION_API aion_status aion_kv8_read(const aion_kv8* kv, int32_t layer, void* k, void* v, int32_t type,
                                              int64_t k_stride, int64_t v_stride, const int32_t* seqs,
                                              const int32_t* pos0, const int32_t* cu, int32_t n_seq, int32_t n_tok,
                                              void* stream) {
    const char* what = "aion_kv8_read";
    aion_status s = check_rows(kv, layer, type, seqs, pos0, cu, n_seq, n_tok, what);
    const int64_t width = s == AION_OK ? (int64_t)kv->n_kv_heads * kv->head_size : 0;
    if (s == AION_OK && k) s = check_matrix(k, k_stride, width, type, n_tok, "k", what);
    if (s == AION_OK && v) s = check_matrix(v, v_stride, width, type, n_tok, "v", what);
    if (s != AION_OK || n_tok == 0 || n_seq == 0 || (!k && !v)) return s;
    DeviceGuard dev(kv->device);
    KV_CUDA(dev.err);
    KvReadArgs a;
    a.c = view_of(kv);
    a.r = {seqs, pos0, cu, n_seq, n_tok};
    a.layer = layer;
    a.k = k;
    a.v = v;
    a.k_stride = k_stride;
    a.v_stride = v_stride;
    a.vec = (!k || vectors(k, k_stride, type)) && (!v || vectors(v, v_stride, type));
    KV_CUDA(type == AION_F32 ? launch_read<float>(a, (cudaStream_t)stream)
            : type == AION_F16 ? launch_read<__half>(a, (cudaStream_t)stream)
                               : launch_read<__nv_bfloat16>(a, (cudaStream_t)stream));
    return AION_OK;
}

// ---------------------------------------------------------------------------
// Attention
// ---------------------------------------------------------------------------
// Which kernel.  k_kv_attention streams a sequence's keys once for each 8 rows
// of a K/V head (rows: tokens x query heads), spread over the whole card;
// k_kv_prompt once for each 256 rows, from one SM.  Per 64 keys the first takes
// the SM about 0.4 us a unit of 8 rows, the second 1.3 to 2.2 us a block of
// 256, whatever there is in it, so the tiles win from about 4 units an SM and
// wave of blocks on.  Measured, us of tiles / of streams, hd 128, page 64:
//   fp32, 32 K/V heads, 4 x 4096 keys   16 rows 127 / 75, 32: 127 / 118, 64: 135 / 212
//   bf16, 8 K/V heads, 16 x 4096 keys   16 rows 100 / 75, 32: 99 / 113, 64: 100 / 200
//   bf16, 8 K/V heads, 1 x 32768 keys   256 rows 713 / 335, 512: 744 / 641, 1024: 748 / 1254
// and within 5% (32768 keys), 14% (4096) and 18% (512) of the better one over 147 such shapes, of equally many rows
// and keys a sequence.  The host knows a call's rows and sequences, not which sequence has how many: a call that mixes
// a long chunk with single rows has one kernel for both, by the average: bf16, 8 K/V heads, 31 rows over 8192 keys and
// a chunk of 512 take 525 us, in calls of their own 116 and 217.
constexpr int kTileUnits = 4;
static bool attention_tiles(const aion_kv8* kv, int n_seq, int n_tok, int group) {
    const int64_t rows = ((int64_t)n_tok * group + n_seq - 1) / n_seq, lines = (int64_t)n_seq * kv->n_kv_heads;
    const int64_t sms = sm_count(kv->device), waves = (lines * ((rows + 255) / 256) + sms - 1) / sms;
    return lines * ((rows + 7) / 8) >= kTileUnits * sms * waves;
}

// Where a sequence holds at most this many groups of 64 keys, its units go to
// one block whole: no join launch.  us, cut / whole, fp32 steps of full
// sequences: 32 x 32 heads of 128 and 512 keys 48.1 / 43.4, 1024 keys 73.7 /
// 70.5; 6 heads of 48 and 512 keys 15.9 / 13.8, 1024 keys 17.5 / 16.1, 2048
// keys 19.5 / 20.4; 1 x 8 heads of 128 (groups of 4) 1024 keys 19.9 / 18.7,
// 2048 keys 21.5 / 24.6.
constexpr int kWholeGroups = 16;
static bool attention_whole(const aion_kv8* kv) {
    return (int64_t)kv->max_pages * kv->page_tokens <= kWholeGroups * kKvaT;
}

extern "C" AION_API int64_t aion_kv8_attention_workspace(const aion_kv8* kv, int32_t n_heads, int32_t n_seq,
                                                         int32_t n_tok) {
    if (check_shape(kv, "aion_kv8_attention_workspace") != AION_OK) return -1;
    if (n_heads < 1 || n_heads % kv->n_kv_heads || n_seq < 0 || n_tok < 0) return -1;
    return attention_whole(kv) ? 0 : (int64_t)sm_count(kv->device) * 2 * 2 * sizeof(KvPart);   // two blocks an SM at most
}

template <typename T, int HDP, int D, bool WIDE>
static cudaError_t launch_attention(KvAttnArgs a, int dev, cudaStream_t st) {
    using SH = KvaShape<HDP, D, WIDE>;
    static std::atomic<uint64_t> opted{0};   // devices whose shared-memory limit is raised
    const uint64_t bit = dev >= 0 && dev < 64 ? 1ull << dev : 0;
    if (!bit || !(opted.load() & bit)) {
        const cudaError_t e = cudaFuncSetAttribute(k_kv_attention<T, HDP, D, WIDE>,
                                                   cudaFuncAttributeMaxDynamicSharedMemorySize, SH::kTotal);
        if (e != cudaSuccess) return e;
        opted.fetch_or(bit);
    }
    a.unit_log = SH::kUnitLog;
    const int blocks = sm_count(dev) * SH::kBlocks;
    k_kv_attention<T, HDP, D, WIDE><<<blocks, kKvaThreads, SH::kTotal, st>>>(a);
    cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess && !a.whole && blocks > 1)
        e = launch_pdl(k_kv_attention_join<T>, dim3(blocks - 1), dim3(kKvJoinThreads), 0, st, a, blocks);
    return e;
}
template <typename T, int D>
static cudaError_t launch_attention_of(const KvAttnArgs& a, int rows, int dev, cudaStream_t st) {
    // Units of 8 rows, or of 4 (16-bit rows) or 2 (fp32), whose turns are shorter but which read the keys anew.
    // us, wide / narrow, 8 K/V heads, 1 x 32768 keys and 16 x 2048: bf16 4 rows 37.9 / 35.8 and 35.8 / 33.8, 5 rows
    // 38.3 / 40.0 and 37.9 / 39.9, 8 rows 37.9 / 39.6 and 37.6 / 39.9, 16 rows 44.0 / 52.2 and 46.1 / 55.0; fp32 2 rows
    // 37.9 / 33.9 and 35.8 / 31.7, 3 rows 37.9 / 38.1 and 35.9 / 37.9, 8 rows 38.1 / 50.2 and 37.0 / 52.2.
    const bool wide = rows > (D == 2 ? 4 : 2);
    if (a.c.hd > 64) return wide ? launch_attention<T, 128, D, true>(a, dev, st) : launch_attention<T, 128, D, false>(a, dev, st);
    return wide ? launch_attention<T, 64, D, true>(a, dev, st) : launch_attention<T, 64, D, false>(a, dev, st);
}

template <typename T>
static cudaError_t launch_prompt(const KvAttnArgs& a, int dev, cudaStream_t st) {
    static std::atomic<uint64_t> opted{0};
    const uint64_t bit = dev >= 0 && dev < 64 ? 1ull << dev : 0;
    if (!bit || !(opted.load() & bit)) {
        const cudaError_t e =
            cudaFuncSetAttribute(k_kv_prompt<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, kKvpSmem);
        if (e != cudaSuccess) return e;
        opted.fetch_or(bit);
    }
    const int64_t blocks = ((int64_t)a.r.n_tok * a.group / 256 + a.r.n_seq) * a.c.nkv;
    k_kv_prompt<T><<<(unsigned)blocks, kKvpThreads, kKvpSmem, st>>>(a);
    return cudaGetLastError();
}

extern "C" AION_API aion_status aion_kv8_attention(const aion_kv8* kv, int32_t layer, const void* q, void* out,
                                                   int32_t type, int32_t n_heads, int64_t q_stride, int64_t out_stride,
                                                   float scale, const int32_t* seqs, const int32_t* pos0,
                                                   const int32_t* cu, int32_t n_seq, int32_t n_tok, void* workspace,
                                                   int64_t workspace_bytes, void* stream) {
    const char* what = "aion_kv8_attention";
    aion_status s = check_rows(kv, layer, type, seqs, pos0, cu, n_seq, n_tok, what);
    if (s != AION_OK) return s;
    if (n_heads < 1 || n_heads % kv->n_kv_heads || (int64_t)n_tok * (n_heads / kv->n_kv_heads) > (1 << 30) ||
        ((int64_t)n_tok * n_heads / 256 + (int64_t)(n_seq + 1) * kv->n_kv_heads) >> 31) {
        aion_thread_error("%s: %d query heads for %d K/V heads, %d rows", what, n_heads, kv->n_kv_heads, n_tok);
        return AION_ERR_SHAPE;
    }
    const int64_t width = (int64_t)n_heads * kv->head_size;
    s = check_matrix(q, q_stride, width, type, n_tok, "q", what);
    if (s == AION_OK) s = check_matrix(out, out_stride, width, type, n_tok, "out", what);
    if (s != AION_OK) return s;
    KV_ARG(isfinite(scale), "%s: the scale is not finite", what);
    if (n_tok == 0 || n_seq == 0) return AION_OK;
    const int64_t el = type_bytes(type), last = n_tok - 1;
    const char *q0 = (const char*)q, *q1 = q0 + (last * q_stride + width) * el;
    const char *o0 = (const char*)out, *o1 = o0 + (last * out_stride + width) * el;
    KV_ARG(q1 <= o0 || o1 <= q0, "%s: q and out overlap", what);
    const bool tiles = attention_tiles(kv, n_seq, n_tok, n_heads / kv->n_kv_heads);
    const int64_t need = tiles ? 0 : aion_kv8_attention_workspace(kv, n_heads, n_seq, n_tok);
    KV_ARG(need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0),
           "%s: needs %lld bytes of 16-byte aligned workspace, got %lld", what, (long long)need,
           (long long)(workspace ? workspace_bytes : 0));
    DeviceGuard dev(kv->device);
    KV_CUDA(dev.err);
    KvAttnArgs a;
    a.c = view_of(kv);
    a.r = {seqs, pos0, cu, n_seq, n_tok};
    a.layer = layer;
    a.n_heads = n_heads;
    a.group = n_heads / kv->n_kv_heads;
    a.q = q;
    a.out = out;
    a.q_stride = q_stride;
    a.out_stride = out_stride;
    a.scale = (scale == 0.0f ? 1.0f / sqrtf((float)kv->head_size) : scale) * 1.4426950408889634f;
    a.vec_q = vectors(q, q_stride, type);
    a.vec_out = vectors(out, out_stride, type);
    a.whole = attention_whole(kv);
    a.parts = (KvPart*)workspace;
    a.unit_log = 0;
    const cudaStream_t st = (cudaStream_t)stream;
    if (tiles) {
        if (type == AION_F32) KV_CUDA((launch_prompt<float>(a, kv->device, st)));
        else if (type == AION_F16) KV_CUDA((launch_prompt<__half>(a, kv->device, st)));
        else KV_CUDA((launch_prompt<__nv_bfloat16>(a, kv->device, st)));
        return AION_OK;
    }
    const int rows = (int)(((int64_t)n_tok + n_seq - 1) / n_seq * a.group);   // of a K/V head, on average
    cudaError_t e;
    if (type == AION_F32) e = launch_attention_of<float, 3>(a, rows, kv->device, st);
    else if (type == AION_F16) e = launch_attention_of<__half, 2>(a, rows, kv->device, st);
    else e = launch_attention_of<__nv_bfloat16, 2>(a, rows, kv->device, st);
    KV_CUDA(e);
    return AION_OK;
}

extern "C" AION_API aion_status aion_kv8_status(const aion_kv8* kv, void* stream) {
    const char* what = "aion_kv8_status";
    const aion_status s = check_cache(kv, what);
    if (s != AION_OK) return s;
    DeviceGuard dev(kv->device);
    KV_CUDA(dev.err);
    const cudaStream_t st = (cudaStream_t)stream;
    KV_CUDA(cudaStreamSynchronize(st));
    // Calls on other streams may record something at any time, so the word is taken in one piece; one call at a time
    // brings what it took to the host.
    static std::mutex one;
    int32_t word = 0;
    {
        const std::lock_guard<std::mutex> hold(one);
        k_kv_take_status<<<1, 1, 0, st>>>(view_of(kv));
        KV_CUDA(cudaGetLastError());
        KV_CUDA(cudaMemcpyAsync(&word, kv->work + 3, 4, cudaMemcpyDeviceToHost, st));
        KV_CUDA(cudaStreamSynchronize(st));
    }
    if (!word) return AION_OK;
    aion_thread_error("%s:%s%s%s%s", what, word & KV_TIMEOUT ? " a bounded device-side wait gave up: its result is invalid;" : "",
                      word & KV_BAD_ARG ? " an entry was out of range or a slot appeared twice;" : "",
                      word & KV_BAD_PAGE ? " a page was missing, or an append met a page that is not its slot's alone;" : "",
                      word & KV_NO_PAGES ? " not enough free pages for an entry of aion_kv8_grow;" : "");
    return word & KV_TIMEOUT ? AION_ERR_TIMEOUT : word & KV_BAD_ARG ? AION_ERR_ARG : word & KV_BAD_PAGE ? AION_ERR_STATE : AION_ERR_OOM;
}
