// 8-bit paged K/V cache: pages and their holders (grow, fork, trim, compact),
// rows in (append) and out (read).  No counterpart in the reference, whose
// cache is one fp32 array per sequence (src/kernel_simd.c:1006-1007).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "common.cuh"

namespace aion {

constexpr int kKvMaxSeqs = 4096;    // slots of a cache: the duplicate check's table in shared memory
constexpr int kKvMaxList = 1024;    // entries of one page call: one thread each
constexpr int kKvMaxHead = 128;

// Bits of the status word (work[0]).
enum KvStatus : int32_t { KV_NO_PAGES = 1, KV_BAD_ARG = 2, KV_BAD_PAGE = 4, KV_TIMEOUT = 8 };

// The cache as kernels take it (aion_kv8 of include/aion.h).
struct KvView {
    int8_t *k, *v;
    float *k_scale, *v_scale;
    int32_t *tables, *lens, *refs, *work;
    int n_layers, n_pages, nkv, page, page_log, hd, max_seqs, max_pages;
    __host__ __device__ long long plane() const { return (long long)n_pages * nkv * page * hd; }   // one layer, K or V
    // work[]: 0 status, 1 moves, 2 pages in use, then three lists of n_pages
    __device__ int32_t* list(int i) const { return work + 4 + (size_t)i * n_pages; }
};

__device__ __forceinline__ void kv_flag(const KvView& c, int bit) { atomicOr(c.work, bit); }

// ---------------------------------------------------------------------------
// Pages.  The lists are short (one thread or one block an entry) and the page
// table of a cache is small, so these kernels are bound by their launch and a
// few dependent trips to L2; only the page copies move bytes.
// ---------------------------------------------------------------------------

// Exclusive scan over the block's 1024 threads; *total in every thread.
__device__ __forceinline__ int block_scan_1024(int v, int* total, int* red) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();   // red may still be read from the last scan
    if (lane == 31) red[warp] = x;
    __syncthreads();
    const int w = red[lane];
    int s = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += y;
    }
    *total = __shfl_sync(0xffffffffu, s, 31);
    const int before = __shfl_sync(0xffffffffu, s - w, warp);
    return before + x - v;
}

// One block.  Thread i takes entry i: what it needs, then an inclusive scan of
// the needs gives its place in the list of free pages; a sweep over refs in
// tiles of 4096 pages builds that list and stops once it is long enough.
__global__ void __launch_bounds__(1024) k_kv_grow(KvView c, const int32_t* seqs, const int32_t* n_new, int n,
                                                  int32_t* pos0) {
    __shared__ int first[kKvMaxSeqs];
    __shared__ int s_upto[kKvMaxList], s_slot[kKvMaxList], s_have[kKvMaxList], s_last[kKvMaxList];
    __shared__ int red[32], s_moves;
    const int i = threadIdx.x;
    for (int j = i; j < c.max_seqs; j += 1024) first[j] = 0x7FFFFFFF;
    if (i == 0) s_moves = 0;
    __syncthreads();
    const int slot = i < n ? seqs[i] : -1;
    bool ok = slot >= 0 && slot < c.max_seqs;
    if (ok) atomicMin(&first[slot], i);
    __syncthreads();
    ok = ok && first[slot] == i;
    const int nn = i < n ? n_new[i] : 0;
    const int old = ok ? c.lens[slot] : 0;
    ok = ok && nn >= 0 && old >= 0 && (long long)old + nn <= (long long)c.max_pages << c.page_log;
    int need = 0, have = 0, last = -1;   // last: the shared last page that gets a copy
    if (ok) {
        have = (old + c.page - 1) >> c.page_log;
        need = ((old + nn + c.page - 1) >> c.page_log) - have;
        if (nn > 0 && (old & (c.page - 1))) {
            const int p = c.tables[(size_t)slot * c.max_pages + have - 1];
            if (p < 0 || p >= c.n_pages) {
                ok = false;
                need = 0;
            } else if (c.refs[p] > 1) {
                last = p;
                need++;
            }
        }
    }
    if (i < n && !ok) kv_flag(c, KV_BAD_ARG);
    int total;
    const int upto = block_scan_1024(need, &total, red) + need;
    s_upto[i] = upto;
    s_slot[i] = slot;
    s_have[i] = have;
    s_last[i] = last;
    // The lowest free pages, as many as are asked for.
    int32_t* list = c.list(2);
    int found = 0;
    for (int base = 0; base < c.n_pages && found < total; base += 4096) {
        int free[4], cnt = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int p = base + 4 * i + e;
            free[e] = p < c.n_pages && c.refs[p] == 0;
            cnt += free[e];
        }
        int tile;
        int at = found + block_scan_1024(cnt, &tile, red);
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (free[e]) list[at++] = base + 4 * i + e;
        found += tile;
    }
    __syncthreads();   // the list and the entries' records are complete
    const int give = min(found, total);
    for (int k = i; k < give; k += 1024) {
        int lo = 0, hi = n - 1;   // the first entry with upto > k
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (s_upto[mid] > k) hi = mid;
            else lo = mid + 1;
        }
        if (s_upto[lo] > found) continue;   // refused: not all of its pages are there
        const int before = lo ? s_upto[lo - 1] : 0, page = list[k];
        int32_t* row = c.tables + (size_t)s_slot[lo] * c.max_pages + s_have[lo];
        const int copy = s_last[lo] >= 0;
        if (copy && k == before) {
            const int m = atomicAdd(&s_moves, 1);
            c.list(0)[m] = s_last[lo];
            c.list(1)[m] = page;
            atomicSub(&c.refs[s_last[lo]], 1);
            row[-1] = page;
        } else {
            row[k - before - copy] = page;
        }
        c.refs[page] = 1;
    }
    const bool granted = ok && upto <= found;
    if (i < n) {
        if (ok && !granted && need > 0) kv_flag(c, KV_NO_PAGES);
        const bool yes = granted || (ok && need == 0);
        if (yes) c.lens[slot] = old + nn;
        pos0[i] = yes ? old : -1;
    }
    __syncthreads();
    if (i == 0) c.work[1] = s_moves;
}

// Gives up pages [stay, have) of a slot's row; the block shares the row.
__device__ __forceinline__ void kv_drop(const KvView& c, int32_t* row, int stay, int have) {
    for (int j = stay + threadIdx.x; j < have; j += blockDim.x) {
        const int p = row[j];
        if (p >= 0 && p < c.n_pages) atomicSub(&c.refs[p], 1);
        row[j] = -1;
    }
}

// Block i takes entry i; every block reads the whole list for the checks.
__global__ void __launch_bounds__(128) k_kv_fork(KvView c, const int32_t* src, const int32_t* dst, const int32_t* keep,
                                                 int n) {
    const int i = blockIdx.x, s = src[i], d = dst[i], want = keep ? keep[i] : 0x7FFFFFFF;
    bool bad = s < 0 || s >= c.max_seqs || d < 0 || d >= c.max_seqs || want < 0;
    for (int j = threadIdx.x; j < n; j += blockDim.x) bad = bad || src[j] == d || (j < i && dst[j] == d);
    if (__syncthreads_or(bad)) {
        if (threadIdx.x == 0) kv_flag(c, KV_BAD_ARG);
        return;
    }
    const int len = min(max(c.lens[s], 0), want), cap = c.max_pages;
    const int used = min((len + c.page - 1) >> c.page_log, cap);
    const int had = min((max(c.lens[d], 0) + c.page - 1) >> c.page_log, cap);
    const int32_t* from = c.tables + (size_t)s * cap;
    int32_t* row = c.tables + (size_t)d * cap;
    kv_drop(c, row, 0, had);
    __syncthreads();   // the row is given up before it is written (also orders the reads of lens[d])
    for (int j = threadIdx.x; j < used; j += blockDim.x) {
        const int p = from[j];
        if (p >= 0 && p < c.n_pages) atomicAdd(&c.refs[p], 1);
        row[j] = p;
    }
    if (threadIdx.x == 0) c.lens[d] = len;
}

__global__ void __launch_bounds__(128) k_kv_trim(KvView c, const int32_t* seqs, const int32_t* keep, int n) {
    const int i = blockIdx.x, s = seqs[i], want = keep ? keep[i] : 0;
    bool bad = s < 0 || s >= c.max_seqs || want < 0;
    for (int j = threadIdx.x; j < i; j += blockDim.x) bad = bad || seqs[j] == s;
    if (__syncthreads_or(bad)) {
        if (threadIdx.x == 0) kv_flag(c, KV_BAD_ARG);
        return;
    }
    const int old = max(c.lens[s], 0), len = min(old, want);
    __syncthreads();   // every thread has the old length
    kv_drop(c, c.tables + (size_t)s * c.max_pages, (len + c.page - 1) >> c.page_log,
            min((old + c.page - 1) >> c.page_log, c.max_pages));
    if (threadIdx.x == 0) c.lens[s] = len;
}

// One block: counts the pages in use, then pairs the used pages behind that
// count with the free ones before it, both in order.
__global__ void __launch_bounds__(1024) k_kv_compact(KvView c, int32_t* n_used) {
    __shared__ int red[32];
    const int i = threadIdx.x;
    int cnt = 0;
    for (int p = i; p < c.n_pages; p += 1024) cnt += c.refs[p] > 0;
    int used;
    block_scan_1024(cnt, &used, red);
    int lows = 0, highs = 0;
    for (int base = 0; base < c.n_pages; base += 4096) {
        int take[4], t = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int p = base + 4 * i + e;
            const int r = p < c.n_pages ? c.refs[p] : 0;
            // low half of the word: free places before U; high half: pages to move
            take[e] = p >= c.n_pages ? 0 : p < used ? (r > 0 ? 0 : 1) : (r > 0 ? 1 << 16 : 0);
            t += take[e];
        }
        int tile;
        int at = block_scan_1024(t, &tile, red);   // at most 4096 a half: the halves do not meet
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int p = base + 4 * i + e;
            if (take[e] == 1) c.list(1)[lows + (at & 0xFFFF)] = p;
            if (take[e] == 1 << 16) c.list(0)[highs + (at >> 16)] = p;
            at += take[e];
        }
        lows += tile & 0xFFFF;
        highs += tile >> 16;
    }
    __syncthreads();
    for (int m = i; m < highs; m += 1024) {   // lows == highs: the pages in use fill 0..U-1
        const int from = c.list(0)[m], to = c.list(1)[m];
        c.refs[to] = c.refs[from];
        c.refs[from] = 0;
        c.list(2)[from] = to;
    }
    if (i == 0) {
        c.work[1] = highs;
        c.work[2] = used;
        if (n_used) *n_used = used;
    }
}

// Copies the pages of lists 0 -> 1 (work[1] of them) in every layer, K and V
// values and scales; with `tables`, rewrites the page tables after a
// compaction.  A unit is 16 KB of one plane of one page: four 16-byte loads in
// flight a thread.
constexpr int kKvCopyThreads = 256, kKvCopyUnit = 4 * 16 * kKvCopyThreads;
__global__ void __launch_bounds__(kKvCopyThreads) k_kv_move(KvView c, int tables) {
    pdl_wait();
    const int moves = c.work[1];
    const long long bytes = (long long)c.nkv * c.page * c.hd;   // one page of one plane
    const int units = (int)((bytes + kKvCopyUnit - 1) / kKvCopyUnit);
    const long long total = (long long)moves * c.n_layers * 2 * units;
    for (long long w = blockIdx.x; w < total; w += gridDim.x) {
        const int u = (int)(w % units);
        const long long r = w / units;
        const int isv = (int)(r & 1), layer = (int)((r >> 1) % c.n_layers), m = (int)((r >> 1) / c.n_layers);
        const int from = c.list(0)[m], to = c.list(1)[m];
        int8_t* pool = (isv ? c.v : c.k) + layer * c.plane();
        const int8_t* s = pool + from * bytes;
        int8_t* d = pool + to * bytes;
        uint4 x[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const long long o = (long long)u * kKvCopyUnit + 16 * (threadIdx.x + e * kKvCopyThreads);
            if (o < bytes) x[e] = *reinterpret_cast<const uint4*>(s + o);
        }
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const long long o = (long long)u * kKvCopyUnit + 16 * (threadIdx.x + e * kKvCopyThreads);
            if (o < bytes) *reinterpret_cast<uint4*>(d + o) = x[e];
        }
        if (u == 0) {
            float* sc = (isv ? c.v_scale : c.k_scale) + (long long)layer * c.n_pages * c.nkv;
            for (int h = threadIdx.x; h < c.nkv; h += kKvCopyThreads)
                sc[(long long)to * c.nkv + h] = sc[(long long)from * c.nkv + h];
        }
    }
    if (!tables || moves == 0) return;
    const int used = c.work[2];
    for (int s = blockIdx.x; s < c.max_seqs; s += gridDim.x) {
        const int len = c.lens[s];
        const int have = len <= 0 ? 0 : min((len + c.page - 1) >> c.page_log, c.max_pages);
        int32_t* row = c.tables + (size_t)s * c.max_pages;
        for (int j = threadIdx.x; j < have; j += kKvCopyThreads) {
            const int p = row[j];
            if (p >= used && p < c.n_pages) row[j] = c.list(2)[p];
        }
    }
}

__global__ void k_kv_reset(KvView c) {
    const long long i0 = blockIdx.x * (long long)blockDim.x + threadIdx.x, step = (long long)gridDim.x * blockDim.x;
    for (long long i = i0; i < c.n_pages; i += step) c.refs[i] = 0;
    for (long long i = i0; i < (long long)c.max_seqs * c.max_pages; i += step) c.tables[i] = -1;
    for (long long i = i0; i < c.max_seqs; i += step) c.lens[i] = 0;
    if (i0 < 4) c.work[i0] = 0;
}

// ---------------------------------------------------------------------------
// Rows of a call: sequence i has rows cu[i]..cu[i+1]-1 at positions pos0[i]...
// ---------------------------------------------------------------------------
struct KvRows {
    const int32_t *seqs, *pos0, *cu;
    int n_seq, n_tok;
    __device__ __forceinline__ int begin(int i) const { return cu ? cu[i] : i; }
    __device__ __forceinline__ int end(int i) const { return cu ? cu[i + 1] : i + 1; }
};

// Blocks of `1 << log` rows or positions are dealt out without a pass over the
// lengths: sequence i has the virtual places (cu[i] >> log) + extra * i and
// on, up to the next one's.  Its cnt = cu[i+1] - cu[i] rows need at most
// (cnt >> log) + extra blocks, and floor(a + b) - floor(a) >= floor(b), so the
// places suffice: extra 1 for blocks of rows, 2 for pages (the first page may
// begin anywhere).  Returns the sequence of place u.
__device__ __forceinline__ int kv_seq_of(const KvRows& r, int u, int log, int extra, int* index) {
    if (!r.cu) {
        *index = 0;
        return u;
    }
    int lo = 0, hi = r.n_seq - 1;   // the last sequence whose first place is <= u
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if ((r.cu[mid] >> log) + extra * mid <= u) lo = mid;
        else hi = mid - 1;
    }
    *index = u - ((r.cu[lo] >> log) + extra * lo);
    return lo;
}
// Places of a call (an upper bound the host knows).
__host__ __device__ inline int kv_places(bool cu, int n_seq, int n_tok, int log, int extra) {
    return cu ? (n_tok >> log) + extra * n_seq : n_seq;
}

template <typename T> __device__ __forceinline__ float to_f32(T x);
template <> __device__ __forceinline__ float to_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ float to_f32<__half>(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// 16 consecutive values; `vec`: the address is 16-byte aligned.
template <typename T>
__device__ __forceinline__ void load16(const T* p, bool vec, float (&x)[16]) {
    T t[16];
    if (vec) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T); i++) reinterpret_cast<uint4*>(t)[i] = reinterpret_cast<const uint4*>(p)[i];
    } else {
#pragma unroll
        for (int i = 0; i < 16; i++) t[i] = p[i];
    }
#pragma unroll
    for (int i = 0; i < 16; i++) x[i] = to_f32(t[i]);
}
template <typename T>
__device__ __forceinline__ void store16(T* p, bool vec, const float (&x)[16]) {
    T t[16];
#pragma unroll
    for (int i = 0; i < 16; i++) t[i] = from_f32<T>(x[i]);
    if (vec) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T); i++) reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(t)[i];
    } else {
#pragma unroll
        for (int i = 0; i < 16; i++) p[i] = t[i];
    }
}

// The integer nearest to the exact x / s (ties to even), within +-127; s > 0.
// The rounded quotient can only be off next to a border between two integers;
// x - q s is exact there (a multiple of the smaller ulp, below 2^24 of them),
// so one fma settles it.
__device__ __forceinline__ int kv_quant(float x, float s) {
    float q = rintf(__fdiv_rn(x, s));
    const float r = 2.0f * __fmaf_rn(-q, s, x);
    q += r > s ? 1.0f : r < -s ? -1.0f : 0.0f;
    return (int)fminf(fmaxf(q, -127.0f), 127.0f);
}
// An earlier value under a page's grown scale.
__device__ __forceinline__ int kv_requant(int q, float ratio) { return (int)rintf((float)q * ratio); }

__device__ __forceinline__ uint32_t pack4(int a, int b, int c, int d) {
    return (a & 0xFF) | (b & 0xFF) << 8 | (c & 0xFF) << 16 | (uint32_t)d << 24;
}

struct KvAppendArgs {
    KvView c;
    KvRows r;
    int layer;
    const void *k, *v;
    long long k_stride, v_stride;
    int vec;
};
// Block (place, head, K or V): the rows of one page and head.
constexpr int kKvAppendThreads = 128;
template <typename T>
__global__ void __launch_bounds__(kKvAppendThreads) k_kv_append(KvAppendArgs a) {
    __shared__ float red[kKvAppendThreads / 32];
    const KvView& c = a.c;
    int idx;
    const int s = kv_seq_of(a.r, blockIdx.x, c.page_log, 2, &idx), h = blockIdx.y, isv = blockIdx.z;
    const int t0 = a.r.begin(s), t1 = min(a.r.end(s), a.r.n_tok), p0 = a.r.pos0[s], slot = a.r.seqs[s];
    if (p0 < 0 || t1 <= t0) return;
    const int pg = (p0 >> c.page_log) + idx;                        // page of the slot
    const long long lo = max((long long)p0, (long long)pg << c.page_log);
    const long long hi = min((long long)p0 + (t1 - t0), (long long)(pg + 1) << c.page_log);
    if (lo >= hi) return;
    bool bad = t0 < 0 || slot < 0 || slot >= c.max_seqs;
    for (int j = threadIdx.x; j < s; j += kKvAppendThreads) bad = bad || a.r.seqs[j] == slot;
    if (__syncthreads_or(bad)) {
        if (threadIdx.x == 0) kv_flag(c, KV_BAD_ARG);
        return;
    }
    const int page = pg < c.max_pages ? c.tables[(size_t)slot * c.max_pages + pg] : -1;
    if (page < 0 || page >= c.n_pages || c.refs[page] != 1) {
        if (threadIdx.x == 0) kv_flag(c, KV_BAD_PAGE);
        return;
    }
    const T* x = (isv ? (const T*)a.v + (t0 + (lo - p0)) * a.v_stride : (const T*)a.k + (t0 + (lo - p0)) * a.k_stride) +
                 (long long)h * c.hd;
    const long long stride = isv ? a.v_stride : a.k_stride;
    const int rows = (int)(hi - lo), row0 = (int)(lo & (c.page - 1)), cpr = c.hd / 16;   // 16-value chunks a row
    int8_t* pool = (isv ? c.v : c.k) + a.layer * c.plane() + ((long long)page * c.nkv + h) * c.page * c.hd;
    float* scale = (isv ? c.v_scale : c.k_scale) + ((long long)a.layer * c.n_pages + page) * c.nkv + h;
    float m = 0.0f;   // NaN once a value is not finite: max() below keeps it
    for (int i = threadIdx.x; i < rows * cpr; i += kKvAppendThreads) {
        float v[16];
        load16(x + (i / cpr) * stride + (i % cpr) * 16, a.vec, v);
#pragma unroll
        for (int e = 0; e < 16; e++) {
            const float b = fabsf(v[e]);
            m = b <= 3.402823466e38f ? fmaxf(m, b) : INFINITY;
        }
    }
    m = warp_max(m);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
    __syncthreads();
    m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float need = m <= 3.402823466e38f ? __fdiv_rn(m, 127.0f) : __int_as_float(0x7FC00000);
    const float s0 = row0 ? *scale : 0.0f;
    float sc = need;
    if (row0 && need <= s0) sc = s0;
    else if (row0 && need == need && s0 == s0) sc = fmaxf(need, 1.25f * s0);
    else if (row0) sc = __int_as_float(0x7FC00000);
    __syncthreads();   // every thread has the old scale
    if (threadIdx.x == 0) *scale = sc;
    if (row0 && sc != s0) {   // also a NaN scale: the earlier values become 0
        const float ratio = sc > 0.0f ? __fdiv_rn(s0, sc) : 0.0f;
        for (int i = threadIdx.x; i < row0 * cpr; i += kKvAppendThreads) {
            uint4* at = reinterpret_cast<uint4*>(pool) + i;
            uint4 w = *at;
            uint32_t* u = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
            for (int e = 0; e < 4; e++)
                u[e] = pack4(kv_requant((int8_t)u[e], ratio), kv_requant((int8_t)(u[e] >> 8), ratio),
                             kv_requant((int8_t)(u[e] >> 16), ratio), kv_requant((int8_t)(u[e] >> 24), ratio));
            *at = w;
        }
    }
    for (int i = threadIdx.x; i < rows * cpr; i += kKvAppendThreads) {
        float v[16];
        load16(x + (i / cpr) * stride + (i % cpr) * 16, a.vec, v);
        int q[16];
#pragma unroll
        for (int e = 0; e < 16; e++) q[e] = sc > 0.0f ? kv_quant(v[e], sc) : 0;
        uint4 w;
        w.x = pack4(q[0], q[1], q[2], q[3]);
        w.y = pack4(q[4], q[5], q[6], q[7]);
        w.z = pack4(q[8], q[9], q[10], q[11]);
        w.w = pack4(q[12], q[13], q[14], q[15]);
        *(reinterpret_cast<uint4*>(pool) + row0 * cpr + i) = w;
    }
}

struct KvReadArgs {
    KvView c;
    KvRows r;
    int layer;
    void *k, *v;
    long long k_stride, v_stride;
    int vec;
};
// Block (place of 32 rows, head): 16 values a thread and step, K then V.
constexpr int kKvReadThreads = 128, kKvReadLog = 5;
template <typename T>
__global__ void __launch_bounds__(kKvReadThreads) k_kv_read(KvReadArgs a) {
    const KvView& c = a.c;
    int idx;
    const int s = kv_seq_of(a.r, blockIdx.x, kKvReadLog, 1, &idx), h = blockIdx.y;
    const int t0 = a.r.begin(s), t1 = min(a.r.end(s), a.r.n_tok), p0 = a.r.pos0[s], slot = a.r.seqs[s];
    const int i0 = idx << kKvReadLog, rows = min(t1 - t0 - i0, 1 << kKvReadLog), cpr = c.hd / 16;
    if (rows <= 0 || t0 < 0) return;
    const bool held = slot >= 0 && slot < c.max_seqs;
    if (!held && p0 >= 0 && threadIdx.x == 0) kv_flag(c, KV_BAD_ARG);
    for (int i = threadIdx.x; i < 2 * rows * cpr; i += kKvReadThreads) {
        const int isv = i >= rows * cpr, j = i - isv * rows * cpr, row = i0 + j / cpr, ch = j % cpr;
        T* out = isv ? (T*)a.v : (T*)a.k;
        if (!out) continue;
        float x[16];
#pragma unroll
        for (int e = 0; e < 16; e++) x[e] = 0.0f;
        if (held && p0 >= 0) {
            const long long pos = (long long)p0 + row;
            const long long pg = pos >> c.page_log;
            const int page = pg < c.max_pages ? c.tables[(size_t)slot * c.max_pages + pg] : -1;
            if (page >= 0 && page < c.n_pages) {
                const float sc = (isv ? c.v_scale : c.k_scale)[((long long)a.layer * c.n_pages + page) * c.nkv + h];
                const int8_t* pool = (isv ? c.v : c.k) + a.layer * c.plane() +
                                     ((long long)page * c.nkv + h) * c.page * c.hd + (pos & (c.page - 1)) * c.hd + 16 * ch;
                const uint4 w = *reinterpret_cast<const uint4*>(pool);
                const int8_t* b = reinterpret_cast<const int8_t*>(&w);
#pragma unroll
                for (int e = 0; e < 16; e++) x[e] = (float)b[e] * sc;
            } else {
                kv_flag(c, KV_BAD_PAGE);
            }
        }
        store16(out + (t0 + row) * (isv ? a.v_stride : a.k_stride) + (long long)h * c.hd + 16 * ch, a.vec, x);
    }
}

}  // namespace aion
