// 8-bit paged K/V cache: pages and their holders (grow, fork, trim, compact),
// rows in (append) and out (read).  No counterpart in the reference, whose
// cache is one fp32 array per sequence (src/kernel_simd.c:1006-1007).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <type_traits>

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
    // work[]: 0 status, 1 moves, 2 pages in use, 3 status on its way to the host, then three lists of n_pages
    __device__ int32_t* list(int i) const { return work + 4 + (size_t)i * n_pages; }
};

__device__ __forceinline__ void kv_flag(const KvView& c, int bit) { atomicOr(c.work, bit); }

// ---------------------------------------------------------------------------
// Pages.  The lists are short (one thread or one block an entry) and the page
// table of a cache is small, so these kernels are bound by their launch and a
// few dependent trips to L2; only the page copies move bytes.
// ---------------------------------------------------------------------------

// Exclusive scan over the block's 1024 threads; *total in every thread.
template <typename V>
__device__ __forceinline__ V block_scan_1024(V v, V* total, V* red) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    V x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const V y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();   // red may still be read from the last scan
    if (lane == 31) red[warp] = x;
    __syncthreads();
    const V w = red[lane];
    V s = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const V y = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += y;
    }
    *total = __shfl_sync(0xffffffffu, s, 31);
    const V before = __shfl_sync(0xffffffffu, s - w, warp);
    return before + x - v;
}

// One block.  Thread i takes entry i: what it needs, then an inclusive scan of
// the needs gives its place in the list of free pages; a sweep over refs in
// tiles of 4096 pages builds that list and stops once it is long enough.  The
// needs add up past 32 bits (1024 entries of up to 2^26 pages), so they are
// summed in 64; a sum past the number of pages is refused whatever it is.
__global__ void __launch_bounds__(1024) k_kv_grow(KvView c, const int32_t* seqs, const int32_t* n_new, int n,
                                                  int32_t* pos0) {
    __shared__ int first[kKvMaxSeqs];
    __shared__ int s_upto[kKvMaxList], s_slot[kKvMaxList], s_have[kKvMaxList], s_last[kKvMaxList];
    __shared__ int red[32], s_moves;
    __shared__ long long wide[32];
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
    long long asked;
    const int upto = (int)min(block_scan_1024<long long>(need, &asked, wide) + need, c.n_pages + 1LL);
    const int total = (int)min(asked, c.n_pages + 1LL);
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
// flight a thread.  Bound by memory: 0.84 GB of pages (32 layers of 32 heads of
// 128, 64 tokens a page) read and written in 288 us, 5.8 TB/s.
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

__global__ void k_kv_take_status(KvView c) { c.work[3] = atomicExch(c.work, 0); }

// ---------------------------------------------------------------------------
// Rows of a call: sequence i has rows cu[i]..cu[i+1]-1 at positions pos0[i]...
// ---------------------------------------------------------------------------
struct KvRows {
    const int32_t *seqs, *pos0, *cu;
    int n_seq, n_tok;
    __device__ __forceinline__ int begin(int i) const { return cu ? cu[i] : i; }
    __device__ __forceinline__ int end(int i) const { return cu ? cu[i + 1] : i + 1; }
    // entry i writes slot `s`; entries that are skipped (padding) or have no rows do not
    __device__ __forceinline__ bool writes(int i, int s) const { return seqs[i] == s && pos0[i] >= 0 && end(i) > begin(i); }
};

// Records row offsets that fall, are negative or pass the rows of the call:
// thread `i0` of `step` of one block.
__device__ __forceinline__ void kv_vet_rows(const KvView& c, const KvRows& r, int i0, int step) {
    if (!r.cu) return;
    for (int i = i0; i < r.n_seq; i += step) {
        const int b = r.cu[i], e = r.cu[i + 1];
        if (r.pos0[i] >= 0 && (b < 0 || e < b || e > r.n_tok)) kv_flag(c, KV_BAD_ARG);
    }
}

// The last i < n with first(i) <= u, where first does not fall and first(0) <=
// u: by a converged warp, 32 places at a time, since one after the other each
// would be a trip to memory.
template <typename First>
__device__ __forceinline__ int kv_warp_find(int n, long long u, First first) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32, i = lo + (threadIdx.x & 31) * step;
        const unsigned in = __ballot_sync(0xffffffffu, i < hi && first(i) <= u) | 1u;
        lo += (31 - __clz(in)) * step;
        hi = min(lo + step, hi);
    }
    return lo;
}

// Blocks of `1 << log` rows or positions are dealt out without a pass over the
// lengths: sequence i has the virtual places (cu[i] >> log) + extra * i and
// on, up to the next one's.  Its cnt = cu[i+1] - cu[i] rows need at most
// (cnt >> log) + extra blocks, and floor(a + b) - floor(a) >= floor(b), so the
// places suffice: extra 1 for blocks of rows, 2 for pages (the first page may
// begin anywhere).  Returns the sequence of place u; *index < 0: the place lies
// in front of cu[0], which need not be 0, and has nothing to do.
__device__ __forceinline__ int kv_seq_of(const KvRows& r, int u, int log, int extra, int* index) {
    if (!r.cu) {
        *index = 0;
        return u;
    }
    const int lo = kv_warp_find(r.n_seq, u, [&](int i) { return (r.cu[i] >> log) + extra * i; });
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

// Four consecutive values; `vec`: rows start on 16 bytes.
template <typename T>
__device__ __forceinline__ float4 load4(const T* p, bool vec) {
    T t[4];
    if (vec) {
        if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(t) = *reinterpret_cast<const uint4*>(p);
        else *reinterpret_cast<uint2*>(t) = *reinterpret_cast<const uint2*>(p);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) t[i] = p[i];
    }
    return make_float4(to_f32(t[0]), to_f32(t[1]), to_f32(t[2]), to_f32(t[3]));
}
template <typename T>
__device__ __forceinline__ void store4(T* p, bool vec, float4 x) {
    T t[4] = {from_f32<T>(x.x), from_f32<T>(x.y), from_f32<T>(x.z), from_f32<T>(x.w)};
    if (vec) {
        if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(p) = *reinterpret_cast<uint4*>(t);
        else *reinterpret_cast<uint2*>(p) = *reinterpret_cast<uint2*>(t);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) p[i] = t[i];
    }
}

// Two fp32 values in one 64-bit register, for the packed fp32 instructions.
__device__ __forceinline__ uint64_t f2_pack(float x, float y) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ float2 f2_unpack(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t f2_mul(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
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

// Four values under a page's scale s > 0, packed.  q = rint(x (1 / s)) can only
// be off where x - q s, which the fma gives exactly, reaches half a scale:
// those and tiny scales take the exact way.
__device__ __forceinline__ uint32_t kv_quant4(float4 x, float s, float inv) {
    constexpr float kMagic = 12582912.0f;   // 1.5 2^23: the sum's low byte is the integer's
    const uint64_t x01 = f2_pack(x.x, x.y), x23 = f2_pack(x.z, x.w), i2 = f2_pack(inv, inv), s2 = f2_pack(-s, -s);
    const uint64_t up = f2_pack(kMagic, kMagic), down = f2_pack(-kMagic, -kMagic);
    const uint64_t m01 = f2_fma(x01, i2, up), m23 = f2_fma(x23, i2, up);
    const float2 r01 = f2_unpack(f2_fma(f2_add(m01, down), s2, x01)), r23 = f2_unpack(f2_fma(f2_add(m23, down), s2, x23));
    const float h = 0.5f * s;
    const bool close = fabsf(r01.x) >= h || fabsf(r01.y) >= h || fabsf(r23.x) >= h || fabsf(r23.y) >= h;
    const float2 a = f2_unpack(m01), b = f2_unpack(m23);
    if (close || s < 1e-30f) return pack4(kv_quant(x.x, s), kv_quant(x.y, s), kv_quant(x.z, s), kv_quant(x.w, s));
    return __byte_perm(__byte_perm(__float_as_uint(a.x), __float_as_uint(a.y), 0x0040),
                       __byte_perm(__float_as_uint(b.x), __float_as_uint(b.y), 0x0040), 0x5410);
}
// Largest magnitude so far, as bits: a NaN or an infinity stays the largest.
__device__ __forceinline__ uint32_t kv_top4(uint32_t top, float4 x) {
    const uint32_t a = max(__float_as_uint(x.x) & 0x7FFFFFFFu, __float_as_uint(x.y) & 0x7FFFFFFFu);
    const uint32_t b = max(__float_as_uint(x.z) & 0x7FFFFFFFu, __float_as_uint(x.w) & 0x7FFFFFFFu);
    return max(top, max(a, b));
}
// The scale of a page whose new rows reach `top`; `old`: that of its earlier rows, if it has any.
__device__ __forceinline__ float kv_scale_of(uint32_t top, bool held, float old) {
    const float nan = __int_as_float(0x7FC00000);
    const float need = top < 0x7F800000u ? __fdiv_rn(__uint_as_float(top), 127.0f) : nan;
    if (!held) return need;
    if (need <= old) return old;
    return need == need && old == old ? fmaxf(need, 1.25f * old) : nan;
}
// Earlier values of a page under its grown scale: words i0, i0 + step, ... of n.
__device__ __forceinline__ void kv_rescale(int8_t* pool, int n, int i0, int step, float old, float s) {
    const float ratio = s > 0.0f ? __fdiv_rn(old, s) : 0.0f;   // also a NaN scale: the values become 0
    for (int i = i0; i < n; i += step) {
        uint32_t* w = reinterpret_cast<uint32_t*>(pool) + i;
        const uint32_t u = *w;
        *w = pack4(kv_requant((int8_t)u, ratio), kv_requant((int8_t)(u >> 8), ratio), kv_requant((int8_t)(u >> 16), ratio),
                   kv_requant((int8_t)(u >> 24), ratio));
    }
}

struct KvAppendArgs {
    KvView c;
    KvRows r;
    int layer;
    const void *k, *v;
    long long k_stride, v_stride;
    int vec;
};
// Block (place, K or V, head, heads fastest: neighbours read neighbouring
// rows): the rows of one page and head, four values a thread and step, all of
// them loaded before the scale is known and kept in registers (PIECES = page hd
// / (4 THREADS) steps at most).  Bound by memory, and by instructions next to
// it, so warps are few and take many steps: with 256 threads a page of 64 took
// 1.1 times as long (a page of 128 has 256, for the registers).  32 x 512 fp32
// rows of 32 heads of 128 take 128 us, 5.2 TB/s.
constexpr int kKvAppendThreads = 256;
template <typename T, int PIECES, int THREADS>
__global__ void __launch_bounds__(THREADS) k_kv_append(KvAppendArgs a) {
    __shared__ uint32_t red[THREADS / 32];
    const KvView& c = a.c;
    const int h = blockIdx.x % c.nkv, isv = (blockIdx.x / c.nkv) & 1;
    if (blockIdx.x == 0) kv_vet_rows(c, a.r, threadIdx.x, THREADS);
    int idx;
    const int s = kv_seq_of(a.r, blockIdx.x / (2 * c.nkv), c.page_log, 2, &idx);
    if (idx < 0) return;
    const int t0 = a.r.begin(s), t1 = min(a.r.end(s), a.r.n_tok), p0 = a.r.pos0[s], slot = a.r.seqs[s];
    if (p0 < 0 || t1 <= t0 || t0 < 0) return;
    const int pg = (p0 >> c.page_log) + idx;                        // page of the slot
    const long long lo = max((long long)p0, (long long)pg << c.page_log);
    const long long hi = min((long long)p0 + (t1 - t0), (long long)(pg + 1) << c.page_log);
    if (lo >= hi) return;
    // the rows are on their way while the page is looked up and checked
    const long long stride = isv ? a.v_stride : a.k_stride;
    const T* x = (isv ? (const T*)a.v : (const T*)a.k) + (t0 + (lo - p0)) * stride + (long long)h * c.hd;
    const int rows = (int)(hi - lo), row0 = (int)(lo & (c.page - 1)), ppr = c.hd / 4, n = rows * ppr;   // pieces of a row
    float4 v[PIECES];
    uint32_t top = 0;
    const int dr = THREADS / ppr, dc = THREADS - dr * ppr, first = threadIdx.x / ppr;
    auto load = [&](auto vec) {
        int col = threadIdx.x - first * ppr;
        const T* p = x + first * stride + 4 * col;
        const long long step = dr * stride + 4 * dc, wrap = stride - c.hd;
#pragma unroll
        for (int e = 0; e < PIECES; e++) {
            v[e] = (int)threadIdx.x + e * THREADS < n ? load4(p, vec.value) : make_float4(0, 0, 0, 0);
            p += step;
            col += dc;
            if (col >= ppr) {
                col -= ppr;
                p += wrap;
            }
        }
    };
    if (a.vec) load(std::true_type{});
    else load(std::false_type{});
    bool bad = slot < 0 || slot >= c.max_seqs;
    for (int j = threadIdx.x; j < s; j += THREADS) bad = bad || a.r.writes(j, slot);
    const int page = slot >= 0 && slot < c.max_seqs && pg < c.max_pages ? c.tables[(size_t)slot * c.max_pages + pg] : -1;
    if (__syncthreads_or(bad)) {
        if (threadIdx.x == 0) kv_flag(c, KV_BAD_ARG);
        return;
    }
    if (page < 0 || page >= c.n_pages || c.refs[page] != 1) {
        if (threadIdx.x == 0) kv_flag(c, KV_BAD_PAGE);
        return;
    }
    int8_t* pool = (isv ? c.v : c.k) + a.layer * c.plane() + ((long long)page * c.nkv + h) * c.page * c.hd;
    float* scale = (isv ? c.v_scale : c.k_scale) + ((long long)a.layer * c.n_pages + page) * c.nkv + h;
    const float old = row0 ? *scale : 0.0f;
#pragma unroll
    for (int e = 0; e < PIECES; e++) top = kv_top4(top, v[e]);
    top = __reduce_max_sync(0xffffffffu, top);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = top;
    __syncthreads();   // every thread has the old scale, too
#pragma unroll
    for (int w = 0; w < THREADS / 32; w++) top = max(top, red[w]);
    const float sc = kv_scale_of(top, row0 != 0, old);
    if (threadIdx.x == 0) *scale = sc;
    if (row0 && sc != old) kv_rescale(pool, row0 * ppr, threadIdx.x, THREADS, old, sc);
    const float inv = __fdiv_rn(1.0f, sc);
    uint32_t* to = reinterpret_cast<uint32_t*>(pool) + row0 * ppr;
#pragma unroll
    for (int e = 0; e < PIECES; e++) {
        const int i = threadIdx.x + e * THREADS;
        if (i < n) to[i] = sc > 0.0f ? kv_quant4(v[e], sc, inv) : 0u;
    }
}

// One row a sequence: a warp takes a sequence, head, and K or V; lane l has
// dimensions 4 l..+3.  Bound by the trips to memory that depend on one another
// (slot and position, page, its scale); the row is loaded alongside the first.
template <typename T>
__global__ void __launch_bounds__(kKvAppendThreads) k_kv_append_one(KvAppendArgs a) {
    const KvView& c = a.c;
    const int lane = threadIdx.x & 31;
    const long long u = (long long)blockIdx.x * (kKvAppendThreads / 32) + (threadIdx.x >> 5);
    const int h = (int)(u % c.nkv), isv = (int)(u / c.nkv) & 1, s = (int)(u / (2 * c.nkv));
    if (s >= a.r.n_seq) return;
    const int p0 = a.r.pos0[s], slot = a.r.seqs[s];
    const T* x = isv ? (const T*)a.v + s * a.v_stride : (const T*)a.k + s * a.k_stride;
    const float4 v = 4 * lane < c.hd ? load4(x + (long long)h * c.hd + 4 * lane, a.vec) : make_float4(0, 0, 0, 0);
    bool twice = false;
    for (int j = lane; j < s; j += 32) twice = twice || a.r.writes(j, slot);
    if (p0 < 0) return;
    if (__any_sync(0xffffffffu, twice) || slot < 0 || slot >= c.max_seqs) {
        if (lane == 0) kv_flag(c, KV_BAD_ARG);
        return;
    }
    const int pg = p0 >> c.page_log, page = pg < c.max_pages ? c.tables[(size_t)slot * c.max_pages + pg] : -1;
    if (page < 0 || page >= c.n_pages) {
        if (lane == 0) kv_flag(c, KV_BAD_PAGE);
        return;
    }
    const int row0 = p0 & (c.page - 1), ppr = c.hd / 4;
    int8_t* pool = (isv ? c.v : c.k) + a.layer * c.plane() + ((long long)page * c.nkv + h) * c.page * c.hd;
    float* scale = (isv ? c.v_scale : c.k_scale) + ((long long)a.layer * c.n_pages + page) * c.nkv + h;
    const float old = *scale;
    if (c.refs[page] != 1) {
        if (lane == 0) kv_flag(c, KV_BAD_PAGE);
        return;
    }
    const float sc = kv_scale_of(__reduce_max_sync(0xffffffffu, kv_top4(0, v)), row0 != 0, old);
    __syncwarp();   // every lane has the old scale
    if (lane == 0) *scale = sc;
    if (row0 && sc != old) kv_rescale(pool, row0 * ppr, lane, 32, old, sc);
    if (4 * lane < c.hd)
        reinterpret_cast<uint32_t*>(pool)[row0 * ppr + lane] = sc > 0.0f ? kv_quant4(v, sc, __fdiv_rn(1.0f, sc)) : 0u;
}

struct KvReadArgs {
    KvView c;
    KvRows r;
    int layer;
    void *k, *v;
    long long k_stride, v_stride;
    int vec;
};
// One row a sequence: a warp takes a sequence, head, and K or V; lane l has
// dimensions 4 l..+3.
template <typename T>
__global__ void __launch_bounds__(kKvAppendThreads) k_kv_read_one(KvReadArgs a) {
    const KvView& c = a.c;
    const int lane = threadIdx.x & 31;
    const long long u = (long long)blockIdx.x * (kKvAppendThreads / 32) + (threadIdx.x >> 5);
    const int h = (int)(u % c.nkv), isv = (int)(u / c.nkv) & 1, s = (int)(u / (2 * c.nkv));
    T* out = isv ? (T*)a.v : (T*)a.k;
    if (s >= a.r.n_seq || !out) return;
    const int p0 = a.r.pos0[s], slot = a.r.seqs[s];
    const bool held = slot >= 0 && slot < c.max_seqs;
    uint32_t w = 0;
    float sc = 0.0f;
    if (p0 >= 0 && held) {
        const int pg = p0 >> c.page_log, page = pg < c.max_pages ? c.tables[(size_t)slot * c.max_pages + pg] : -1;
        if (page >= 0 && page < c.n_pages) {
            const long long unit = (long long)page * c.nkv + h;
            sc = (isv ? c.v_scale : c.k_scale)[(long long)a.layer * c.n_pages * c.nkv + unit];
            if (4 * lane < c.hd)
                w = *reinterpret_cast<const uint32_t*>((isv ? c.v : c.k) + a.layer * c.plane() +
                                                       (unit * c.page + (p0 & (c.page - 1))) * c.hd + 4 * lane);
        } else if (lane == 0) {
            kv_flag(c, KV_BAD_PAGE);
        }
    } else if (p0 >= 0 && lane == 0) {
        kv_flag(c, KV_BAD_ARG);
    }
    if (4 * lane < c.hd)
        store4(out + s * (isv ? a.v_stride : a.k_stride) + (long long)h * c.hd + 4 * lane, a.vec,
               make_float4((float)(int8_t)w * sc, (float)(int8_t)(w >> 8) * sc, (float)(int8_t)(w >> 16) * sc,
                           (float)(int8_t)(w >> 24) * sc));
}

// Block (place of 64 rows, K or V, head, heads fastest): four values a thread
// and step, eight steps in flight.  Bound by memory, the writes above all: 32 x
// 512 fp32 rows of 32 heads of 128 take 115 us, 5.8 TB/s (127 us in blocks of
// 256 with divisions for each piece).
constexpr int kKvReadThreads = 128, kKvReadLog = 6, kKvReadSteps = 8;
template <typename T>
__global__ void __launch_bounds__(kKvReadThreads) k_kv_read(KvReadArgs a) {
    __shared__ long long s_at[8];
    __shared__ float s_scale[8];
    const KvView& c = a.c;
    const int h = blockIdx.x % c.nkv, isv = (blockIdx.x / c.nkv) & 1;
    T* out = isv ? (T*)a.v : (T*)a.k;
    if (blockIdx.x == 0) kv_vet_rows(c, a.r, threadIdx.x, kKvReadThreads);
    if (!out) return;
    int idx;
    const int s = kv_seq_of(a.r, blockIdx.x / (2 * c.nkv), kKvReadLog, 1, &idx);
    if (idx < 0) return;
    const int t0 = a.r.begin(s), t1 = min(a.r.end(s), a.r.n_tok), p0 = a.r.pos0[s], slot = a.r.seqs[s];
    const int i0 = idx << kKvReadLog, rows = min(t1 - t0 - i0, 1 << kKvReadLog), ppr = c.hd / 4, n = rows * ppr;
    if (rows <= 0 || t0 < 0) return;
    const bool held = slot >= 0 && slot < c.max_seqs;
    if (!held && p0 >= 0 && threadIdx.x == 0) kv_flag(c, KV_BAD_ARG);
    // the pages that the rows lie in: five at most
    const long long first = (long long)p0 + i0, pg0 = first >> c.page_log;
    if (threadIdx.x < 8) {
        const long long pg = pg0 + threadIdx.x;
        long long at = -1;
        float sc = 0.0f;
        if (held && p0 >= 0 && pg <= (first + rows - 1) >> c.page_log) {
            const int page = pg < c.max_pages ? c.tables[(size_t)slot * c.max_pages + pg] : -1;
            if (page < 0 || page >= c.n_pages) {
                kv_flag(c, KV_BAD_PAGE);
            } else {
                const long long unit = (long long)page * c.nkv + h;
                at = a.layer * c.plane() + unit * c.page * c.hd;
                sc = (isv ? c.v_scale : c.k_scale)[(long long)a.layer * c.n_pages * c.nkv + unit];
            }
        }
        s_at[threadIdx.x] = at;
        s_scale[threadIdx.x] = sc;
    }
    __syncthreads();
    const long long stride = isv ? a.v_stride : a.k_stride;
    const int8_t* pool = isv ? c.v : c.k;
    const int in = (int)(first & (c.page - 1));   // the first row's place in its page
    out += (long long)(t0 + i0) * stride + (long long)h * c.hd;
    const int dr = kKvReadThreads / ppr, dc = kKvReadThreads - dr * ppr;   // from a thread's piece to its next
    int row = threadIdx.x / ppr, col = threadIdx.x - row * ppr;
    auto copy = [&](auto vec) {
#pragma unroll 1
        for (int i0 = threadIdx.x; i0 < n; i0 += kKvReadSteps * kKvReadThreads) {
            uint32_t w[kKvReadSteps];
            float sc[kKvReadSteps];
            const int row0 = row, col0 = col;
            auto next = [&] {
                row += dr;
                col += dc;
                if (col >= ppr) {
                    col -= ppr;
                    row++;
                }
            };
#pragma unroll
            for (int e = 0; e < kKvReadSteps; e++, next()) {
                const int r = in + row, pg = r >> c.page_log;
                const bool there = i0 + e * kKvReadThreads < n;
                const long long at = there ? s_at[pg] : -1;
                w[e] = at >= 0 ? *reinterpret_cast<const uint32_t*>(pool + at + (r & (c.page - 1)) * c.hd + 4 * col) : 0u;
                sc[e] = there ? s_scale[pg] : 0.0f;
            }
            row = row0;
            col = col0;
#pragma unroll
            for (int e = 0; e < kKvReadSteps; e++, next())
                if (i0 + e * kKvReadThreads < n)
                    store4(out + row * stride + 4 * col, vec.value,
                           make_float4((float)(int8_t)w[e] * sc[e], (float)(int8_t)(w[e] >> 8) * sc[e],
                                       (float)(int8_t)(w[e] >> 16) * sc[e], (float)(int8_t)(w[e] >> 24) * sc[e]));
        }
    };
    if (a.vec) copy(std::true_type{});
    else copy(std::false_type{});
}

}  // namespace aion
