// Attention over the 8-bit paged K/V cache (kv8.cuh) for few query rows a
// sequence: single tokens, drafts.
#pragma once

#include <stddef.h>

#include "kv8.cuh"

namespace aion {

struct KvAttnArgs {
    KvView c;
    KvRows r;
    int layer, n_heads, group;   // group: query heads of one K/V head
    const void* q;
    void* out;
    long long q_stride, out_stride;
    float scale;                 // of the scores, times log2(e): the softmax is in base 2
    int vec_q, vec_out;          // rows are 16-byte aligned
    int whole;                   // blocks take whole units: nothing is left to join
    struct KvPart* parts;        // [blocks][2], else
};

// ---------------------------------------------------------------------------
// Arithmetic.  K and V stay the int8 values that the cache holds; the query
// and the softmax weights become fixed-point numbers of D base-256 digits, so
// that every product is an exact integer dot on the tensor cores
// (mma.sync.m16n8k32, s32 accumulators):
//   q = rint(x 127 256^(D-1) / max|x|), digits in -128..127, per row;
//   score = max|x| / (127 256^(D-1)) * K scale * sum_d 256^(D-1-d) (K . q_d);
//   w = rint(2^(score - group max) (256^D - 1)), digits in 0..255;
//   out += V scale * 2^(group max - running max) / (256^D - 1) * sum_d ....
// D is 3 for fp32 rows (a step of 2^-23 of the largest value: fp32's own) and
// 2 for 16-bit rows (2^-15, against the 2^-8 or 2^-11 of a rounded result).
// Digits of one row are columns of different MMAs, so a lane joins them
// without an exchange.  Weights are relative to the largest of their 64
// positions, so a position far below its row's maximum keeps its share.  Sums
// run in fp32.
//
// Work.  A unit is (sequence, K/V head, up to 8 rows: tokens x query heads of
// that K/V head); its keys come in groups of 64.  All groups of all units form
// one line that is cut evenly over the blocks and, in a block, over its warps,
// so uneven lengths and one long sequence load the card alike.  A warp streams
// through its stretch, across the borders of units, with copies in flight all
// the time; what it holds of a unit that others share goes into shared memory
// and is joined in order, and what blocks share goes through `parts` to
// k_kv_attention_join.
//
// Memory.  Each warp has a ring of three slots of 64 rows; K and V slots
// alternate, so two slots (16 KB a warp, 128 KB an SM) are in flight while one
// is used.  16 rows of a page and head are contiguous: a lane copies 16-byte
// pieces (cp.async).  K fragments are 16-byte shared-memory reads (the order
// of the dimensions inside a dot is free, as q's digits take the same order);
// V fragments need four tokens of one dimension in a word: four words of four
// tokens, transposed with byte permutes.  The pieces are XOR-swizzled so that
// both reads touch every bank once.
// ---------------------------------------------------------------------------
constexpr int kKvaWarps = 8, kKvaThreads = 32 * kKvaWarps, kKvaT = 64, kKvaRows = 8;

// 2^x to about 2^-22; 0 below the normal range.
__device__ __forceinline__ float kv_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Softmax state of one unit over a stretch of its keys.
struct alignas(16) KvPart {
    long long begin, end, at;    // the unit's groups in the line; the block's first group
    int s, h, rg, valid;
    float m[kKvaRows], l[kKvaRows];
    alignas(16) float o[kKvaRows][kKvMaxHead];
};
static_assert(offsetof(KvPart, o) % 16 == 0 && sizeof(KvPart) % 16 == 0, "partial rows are read as float4");

__device__ __forceinline__ void mma_ss(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_su(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Four words of four bytes, transposed.
__device__ __forceinline__ void transpose4(uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t (&r)[4]) {
    const uint32_t ab0 = __byte_perm(a, b, 0x5140), ab1 = __byte_perm(a, b, 0x7362);
    const uint32_t cd0 = __byte_perm(c, d, 0x5140), cd1 = __byte_perm(c, d, 0x7362);
    r[0] = __byte_perm(ab0, cd0, 0x5410);
    r[1] = __byte_perm(ab0, cd0, 0x7632);
    r[2] = __byte_perm(ab1, cd1, 0x5410);
    r[3] = __byte_perm(ab1, cd1, 0x7632);
}
template <int N> __device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }

template <int D> struct KvDigits {
    static constexpr float kQ = D == 3 ? 127.0f * 65536.0f : 127.0f * 256.0f;
    static constexpr float kP = D == 3 ? 16777215.0f : 65535.0f;
    // sum over the digits of 256^(D-1-d) c[d]; each c[d] is below 2^24
    static __device__ __forceinline__ float join(const int (&c)[D][4], int e) {
        if constexpr (D == 3) return fmaf((float)c[0][e], 65536.0f, fmaf((float)c[1][e], 256.0f, (float)c[2][e]));
        else return fmaf((float)c[0][e], 256.0f, (float)c[1][e]);
    }
};

// What a call says about sequence s.
struct KvSeq {
    int slot, p0, t0, cnt, len, ng, nrg;
};
__device__ __forceinline__ KvSeq kv_seq(const KvAttnArgs& a, int s) {
    KvSeq q;
    q.slot = a.r.seqs[s];
    q.p0 = a.r.pos0[s];
    q.t0 = a.r.begin(s);
    q.cnt = max(min(a.r.end(s), a.r.n_tok) - q.t0, 0);
    if (q.t0 < 0) q.cnt = 0;
    const bool held = q.p0 >= 0 && q.slot >= 0 && q.slot < a.c.max_seqs;
    const long long len = held ? (long long)q.p0 + q.cnt : 0;
    q.len = (int)min(len, (long long)a.c.max_pages << a.c.page_log);
    // a sequence that sees nothing has one group without keys: its rows become zero
    q.ng = q.cnt ? max((q.len + kKvaT - 1) / kKvaT, 1) : 0;
    q.nrg = (q.cnt * a.group + kKvaRows - 1) / kKvaRows;
    return q;
}

// Records what is wrong with a sequence: a slot that does not exist, positions behind its table.
__device__ __forceinline__ void kv_vet_seq(const KvAttnArgs& a, const KvSeq& q) {
    if (q.p0 < 0 || q.cnt == 0) return;
    if (q.slot < 0 || q.slot >= a.c.max_seqs) kv_flag(a.c, KV_BAD_ARG);
    else if ((long long)q.p0 + q.cnt > q.len) kv_flag(a.c, KV_BAD_PAGE);
}

// A place in the line of groups.
struct KvCursor {
    KvSeq q;
    int s, h, rg, g;
    __device__ __forceinline__ void seek(const KvAttnArgs& a, int seq, long long rest) {
        s = seq;
        q = kv_seq(a, s);
        const long long u = rest / q.ng;
        g = (int)(rest - u * q.ng);
        h = (int)(u / q.nrg);
        rg = (int)(u - (long long)h * q.nrg);
    }
    __device__ __forceinline__ void next(const KvAttnArgs& a) {
        if (++g < q.ng) return;
        g = 0;
        if (++rg < q.nrg) return;
        rg = 0;
        if (++h < a.c.nkv) return;
        h = 0;
        do {
            if (++s >= a.r.n_seq) return;   // the line's end: not used any more
            q = kv_seq(a, s);
        } while (q.cnt == 0);
    }
};

template <int HDP> struct KvaSmem {
    static constexpr int kSlot = kKvaT * HDP;
    static constexpr int kRing = 3 * kSlot;
    static constexpr int kPiece = (kKvaRows * HDP + 2 * kKvaRows) * 4;   // o, m, l
    struct Info {   // of a piece; the unit's groups from the block's first one on
        int begin, end, s, h, rg, valid;
    };
    static_assert(kPiece % 16 == 0 && kRing % 16 == 0 && kKvaRows * 68 * 4 <= kSlot, "float4 pieces, the weights' place");
    static constexpr int kInfo = kKvaWarps * kRing + kKvaWarps * kPiece;
    static constexpr int kTotal = kInfo + 2 * kKvaWarps * (int)sizeof(Info);
};

// Rows of a unit as the lanes see them.
struct KvRow {
    long long q, out;   // element offsets
    int lim;            // last position seen; -1: no row
};
__device__ __forceinline__ KvRow kv_row(const KvAttnArgs& a, const KvSeq& q, int h, int rg, int r) {
    KvRow w;
    const int i = rg * kKvaRows + r, tok = i / a.group, head = h * a.group + (i - tok * a.group);
    w.lim = i < q.cnt * a.group ? (int)min((long long)q.p0 + tok, (long long)q.len - 1) : -1;
    w.q = (q.t0 + tok) * a.q_stride + (long long)head * a.c.hd;
    w.out = i < q.cnt * a.group ? (q.t0 + tok) * a.out_stride + (long long)head * a.c.hd : -1;
    return w;
}

template <typename T>
__device__ __forceinline__ void store4(T* p, bool vec, float4 x) {
    if (vec) {
        if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<float4*>(p) = x;
        } else {
            T t[4] = {from_f32<T>(x.x), from_f32<T>(x.y), from_f32<T>(x.z), from_f32<T>(x.w)};
            *reinterpret_cast<uint2*>(p) = *reinterpret_cast<uint2*>(t);
        }
    } else {
        p[0] = from_f32<T>(x.x);
        p[1] = from_f32<T>(x.y);
        p[2] = from_f32<T>(x.z);
        p[3] = from_f32<T>(x.w);
    }
}

template <typename T, int HDP, int D>
__global__ void __launch_bounds__(kKvaThreads, HDP == 64 ? 2 : 1) k_kv_attention(const KvAttnArgs a) {
    using SM = KvaSmem<HDP>;
    using DG = KvDigits<D>;
    constexpr int NW = HDP / 32;    // 32-dimension segments
    constexpr int NP = HDP / 64;    // pairs of k-steps of the score dot
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ long long s_range[2], s_red[kKvaWarps];
    const KvView& c = a.c;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    unsigned char* ring = smem + warp * SM::kRing;
    float* piece0 = reinterpret_cast<float*>(smem + kKvaWarps * SM::kRing + warp * SM::kPiece);
    typename SM::Info* info = reinterpret_cast<typename SM::Info*>(smem + SM::kInfo);

    // ---- the line: prefix sums of the sequences' groups (in the ring's memory), the block's and the warp's stretch
    long long* pre = reinterpret_cast<long long*>(smem);
    const int per = (a.r.n_seq + kKvaThreads - 1) / kKvaThreads, sa = min((int)threadIdx.x * per, a.r.n_seq),
              sb = min(sa + per, a.r.n_seq);
    long long mine = 0;
    for (int s = sa; s < sb; s++) {
        const KvSeq q = kv_seq(a, s);
        if (blockIdx.x == 0) kv_vet_seq(a, q);
        mine += (long long)q.ng * q.nrg * c.nkv;
    }
    long long x = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) s_red[warp] = x;
    __syncthreads();
    long long W = 0, base = 0;
    for (int w = 0; w < kKvaWarps; w++) {
        if (w == warp) base = W;
        W += s_red[w];
    }
    long long run = base + x - mine;
    for (int s = sa; s < sb; s++) {
        pre[s] = run;
        const KvSeq q = kv_seq(a, s);
        run += (long long)q.ng * q.nrg * c.nkv;
    }
    if (threadIdx.x == 0) pre[a.r.n_seq] = W;
    __syncthreads();
    auto find = [&](long long v) {   // the sequence that group v < W lies in
        int lo = 0, hi = a.r.n_seq - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (pre[mid] <= v) lo = mid;
            else hi = mid - 1;
        }
        return lo;
    };
    // a group for each warp at least: few blocks where there is little to do
    const long long nb = min((long long)gridDim.x, (W + kKvaWarps - 1) / kKvaWarps);
    if (threadIdx.x < 2) {
        const long long b = blockIdx.x + threadIdx.x;
        long long v = b >= nb ? W : W * b / nb;
        if (a.whole && v < W) {   // up to the next unit's start
            const int s = find(v);
            const long long ng = kv_seq(a, s).ng, rest = v - pre[s];
            v = pre[s] + (rest + ng - 1) / ng * ng;
        }
        s_range[threadIdx.x] = v;
    }
    __syncthreads();
    const long long b0 = s_range[0], b1 = s_range[1];
    const long long w0 = b0 + (b1 - b0) * warp / kKvaWarps, w1 = b0 + (b1 - b0) * (warp + 1) / kKvaWarps;
    const int n = (int)(w1 - w0);
    KvCursor cur, ahead;   // the group in use; the group whose pages are looked up
    if (n > 0) {
        const int s = find(w0);
        cur.seek(a, s, w0 - pre[s]);
        ahead = cur;
    }
    if (lane < 2) info[2 * warp + lane].valid = 0;
    __syncthreads();   // the ring is free

    // ---- copies
    // A lane's pieces of 16 rows: source 16 (lane + 32 e), destinations swizzled.
    constexpr int NE = HDP / 32;
    int kdst[NE], vdst[NE];
    const int cpr = c.hd / 16;
#pragma unroll
    for (int e = 0; e < NE; e++) {
        const int i = lane + 32 * e, row = i / cpr, ch = i - row * cpr;
        if constexpr (HDP == 128) {
            kdst[e] = row * 128 + (ch ^ (4 * (row & 1))) * 16;
            vdst[e] = row * 128 + ((ch >> 1) ^ ((row >> 2) & 3)) * 32 + (ch & 1) * 16;
        } else {
            kdst[e] = row * 64 + ch * 16;
            vdst[e] = row * 64 + ((ch >> 1) ^ ((row >> 2) & 1)) * 32 + (ch & 1) * 16;
        }
    }
    struct Item {   // pages (lanes 4 i + j: tile j of 16 positions; -1: none), place
        int page, h, g, want;
    };
    auto look = [&](const KvCursor& k) {
        Item it;
        it.h = k.h;
        it.g = k.g;
        it.page = -1;
        const int pos = k.g * kKvaT + 16 * t;
        it.want = pos < k.q.len;
        if (it.want) it.page = c.tables[(size_t)k.q.slot * c.max_pages + (pos >> c.page_log)];
        return it;
    };
    auto vet = [&](Item& it) {   // pages that are missing are left out
        if (it.page < 0 || it.page >= c.n_pages) {
            if (it.want) kv_flag(c, KV_BAD_PAGE);
            it.page = -1;
        }
    };
    auto copy = [&](const Item& it, const int8_t* pool, const int (&dst)[NE], int slot) {
        const uint32_t to = smem_addr(ring + slot * SM::kSlot);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int page = __shfl_sync(0xffffffffu, it.page, j);
            if (page < 0) continue;
            const int8_t* from =
                pool + (((long long)page * c.nkv + it.h) * c.page + ((it.g * kKvaT + 16 * j) & (c.page - 1))) * c.hd;
#pragma unroll
            for (int e = 0; e < NE; e++)
                if (lane + 32 * e < c.hd)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + j * 16 * HDP + dst[e]),
                                 "l"(from + 16 * (lane + 32 * e))
                                 : "memory");
        }
    };
    const int8_t *kp = c.k + a.layer * c.plane(), *vp = c.v + a.layer * c.plane();
    const float* scales = (lane < 4 ? c.k_scale : c.v_scale) + (long long)a.layer * c.n_pages * c.nkv;
    auto scale_of = [&](const Item& it) {   // lanes 0..3: K scales of the tiles, 4..7: V scales
        return it.page >= 0 ? scales[(long long)it.page * c.nkv + it.h] : 0.0f;
    };

    // ---- state of the unit in use
    float o[NW][2][4], m[2], l[2], rs[2];
    int lim[2];
    uint32_t qd[D][NP][4];
    bool fresh = true;   // the unit began in this warp's stretch
    auto begin_unit = [&]() {
#pragma unroll
        for (int w = 0; w < NW; w++)
#pragma unroll
            for (int i = 0; i < 8; i++) o[w][i >> 2][i & 3] = 0.0f;
        m[0] = m[1] = -INFINITY;
        l[0] = l[1] = 0.0f;
        // lane (g, t): row g, dimensions 16 (4 p + t)..+15
        const KvRow row = kv_row(a, cur.q, cur.h, cur.rg, g);
        float v[NP][16], top = 0.0f;
        bool bad = false;
#pragma unroll
        for (int p = 0; p < NP; p++) {
            const int d0 = 16 * (4 * p + t);
            if (row.lim >= 0 && d0 < c.hd) {
                load16((const T*)a.q + row.q + d0, a.vec_q, v[p]);
            } else {
#pragma unroll
                for (int i = 0; i < 16; i++) v[p][i] = 0.0f;
            }
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const float b = fabsf(v[p][i]);
                bad = bad || !(b <= 3.402823466e38f);
                top = fmaxf(top, b);
            }
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const unsigned bads = __ballot_sync(0xffffffffu, bad);
        bad = (bads >> (4 * g)) & 15;
        // rows of tiny values are scaled up first, so that the factor stays finite
        const float up = top < 8.6736174e-19f ? 1.8446744e19f : 1.0f;   // 2^-60, 2^64
        const float f = top > 0.0f && !bad ? DG::kQ / (top * up) : 0.0f;
#pragma unroll
        for (int p = 0; p < NP; p++)
#pragma unroll
            for (int w = 0; w < 4; w++) {
                int d[D][4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    int z = bad ? 0 : __float2int_rn(v[p][4 * w + i] * up * f);
#pragma unroll
                    for (int k = D - 1; k >= 0; k--) {
                        d[k][i] = (int8_t)z;
                        z = (z - d[k][i]) >> 8;
                    }
                }
#pragma unroll
                for (int k = 0; k < D; k++) qd[k][p][w] = pack4(d[k][0], d[k][1], d[k][2], d[k][3]);
            }
        float r = bad ? __int_as_float(0x7FC00000) : top / DG::kQ * a.scale;
        rs[0] = __shfl_sync(0xffffffffu, r, 8 * t);        // rows 2 t, 2 t + 1
        rs[1] = __shfl_sync(0xffffffffu, r, 8 * t + 4);
        lim[0] = __shfl_sync(0xffffffffu, row.lim, 8 * t);
        lim[1] = __shfl_sync(0xffffffffu, row.lim, 8 * t + 4);
    };
    auto sum_l = [&]() {   // the lanes of a row have summed their own positions
#pragma unroll
        for (int e = 0; e < 2; e++) {
            l[e] += __shfl_xor_sync(0xffffffffu, l[e], 4);
            l[e] += __shfl_xor_sync(0xffffffffu, l[e], 8);
            l[e] += __shfl_xor_sync(0xffffffffu, l[e], 16);
        }
    };
    // The unit's sums so far into a piece; `at`: the group in use, from the block's first on.
    auto put_piece = [&](float* p, int which, int at) {
        sum_l();
#pragma unroll
        for (int e = 0; e < 2; e++) {
            float* row = p + (2 * t + e) * HDP;
#pragma unroll
            for (int w = 0; w < NW; w++)
                *reinterpret_cast<float4*>(row + 32 * w + 4 * g) =
                    make_float4(o[w][0][e], o[w][0][2 + e], o[w][1][e], o[w][1][2 + e]);
            if (g == 0) {
                p[kKvaRows * HDP + 2 * t + e] = m[e];
                p[kKvaRows * HDP + kKvaRows + 2 * t + e] = l[e];
            }
        }
        if (lane == 0) info[2 * warp + which] = {at - cur.g, at - cur.g + cur.q.ng, cur.s, cur.h, cur.rg, 1};
    };
    auto put_rows = [&]() {
        sum_l();
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const KvRow row = kv_row(a, cur.q, cur.h, cur.rg, 2 * t + e);
            if (row.out < 0) continue;
            const float inv = l[e] == 0.0f ? 0.0f : 1.0f / l[e];
#pragma unroll
            for (int w = 0; w < NW; w++)
                if (32 * w + 4 * g < c.hd)
                    store4((T*)a.out + row.out + 32 * w + 4 * g, a.vec_out,
                           make_float4(o[w][0][e] * inv, o[w][0][2 + e] * inv, o[w][1][e] * inv, o[w][1][2 + e] * inv));
        }
    };

    if (n > 0) {
        Item i1, i2, i3;      // one, two, three groups ahead of the one in use
        float sc0, sc1, sc2;  // scales of the group in use and the two behind it
        Item i0 = look(ahead);
        vet(i0);
        i1 = i2 = i3 = i0;
        i1.page = i2.page = i3.page = -1;
        if (n > 1) {
            ahead.next(a);
            i1 = look(ahead);
            vet(i1);
        }
        copy(i0, kp, kdst, 0);
        cp_async_commit();
        copy(i0, vp, vdst, 1);
        cp_async_commit();
        copy(i1, kp, kdst, 2);
        cp_async_commit();
        sc0 = scale_of(i0);
        sc1 = scale_of(i1);
        sc2 = 0.0f;
        if (n > 2) {
            ahead.next(a);
            i2 = look(ahead);   // vetted when it is used: the load is on its way
        }
        fresh = cur.g == 0;
        begin_unit();
        int slot = 0;   // of the next K or V rows to be used
        for (int i = 0; i < n; i++) {
            if (i > 0) {
                const bool last = cur.g + 1 == cur.q.ng;
                if (last) {   // the unit ended with the group before
                    if (fresh) put_rows();
                    else put_piece(piece0, 0, (int)(w0 - b0) + i - 1);
                }
                cur.next(a);
                if (last) {
                    fresh = true;
                    begin_unit();
                }
            }
            // ---- scores
            cp_async_wait<2>();
            __syncwarp();
            unsigned char* ks = ring + slot * SM::kSlot;
            const float vs[4] = {__shfl_sync(0xffffffffu, sc0, 4), __shfl_sync(0xffffffffu, sc0, 5),
                                 __shfl_sync(0xffffffffu, sc0, 6), __shfl_sync(0xffffffffu, sc0, 7)};
            const unsigned live = __ballot_sync(0xffffffffu, i0.page >= 0);
            float p[4][4], mg[2] = {-INFINITY, -INFINITY};   // p[tile][e]: positions g, g + 8 (e >> 1), rows 2 t + (e & 1)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                int acc[D][4];
#pragma unroll
                for (int d = 0; d < D; d++) acc[d][0] = acc[d][1] = acc[d][2] = acc[d][3] = 0;
#pragma unroll
                for (int pp = 0; pp < NP; pp++) {
                    const int r0 = 16 * j + g;
                    const int at = HDP == 128 ? r0 * 128 + ((4 * pp + t) ^ (4 * (g & 1))) * 16 : r0 * 64 + t * 16;
                    const uint4 lo = *reinterpret_cast<const uint4*>(ks + at);
                    const uint4 hi = *reinterpret_cast<const uint4*>(ks + at + 8 * HDP);
                    const uint32_t f0[4] = {lo.x, hi.x, lo.y, hi.y}, f1[4] = {lo.z, hi.z, lo.w, hi.w};
#pragma unroll
                    for (int d = 0; d < D; d++) {
                        mma_ss(acc[d], f0, qd[d][pp][0], qd[d][pp][1]);
                        mma_ss(acc[d], f1, qd[d][pp][2], qd[d][pp][3]);
                    }
                }
                const float kscale = __shfl_sync(0xffffffffu, sc0, j);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int pos = cur.g * kKvaT + 16 * j + g + 8 * (e >> 1);
                    const bool see = pos <= lim[e & 1] && ((live >> j) & 1);
                    p[j][e] = see ? DG::join(acc, e) * (rs[e & 1] * kscale) : -INFINITY;
                    mg[e & 1] = fmaxf(mg[e & 1], p[j][e]);
                }
            }
            // ---- weights relative to the group's largest
            float alpha[2], wt[2], vmax = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; j++)
                if ((live >> j) & 1) vmax = fmaxf(vmax, vs[j]);   // without a NaN
#pragma unroll
            for (int e = 0; e < 2; e++) {
                mg[e] = fmaxf(mg[e], __shfl_xor_sync(0xffffffffu, mg[e], 4));
                mg[e] = fmaxf(mg[e], __shfl_xor_sync(0xffffffffu, mg[e], 8));
                mg[e] = fmaxf(mg[e], __shfl_xor_sync(0xffffffffu, mg[e], 16));
                const float mn = fmaxf(m[e], mg[e]);
                alpha[e] = m[e] == -INFINITY ? 0.0f : kv_exp2(m[e] - mn);
                wt[e] = mg[e] == -INFINITY ? 0.0f : kv_exp2(mg[e] - mn);
                m[e] = mn;
            }
            uint32_t* fx = reinterpret_cast<uint32_t*>(ks);   // [row][68]: the K slot is read
            __syncwarp();
            float sum[2] = {0.0f, 0.0f};
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float ratio = DG::kP * (c.page >= kKvaT ? 1.0f : vmax > 0.0f ? vs[j] / vmax : 0.0f);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const bool none = p[j][e] == -INFINITY;
                    const float w = none ? 0.0f : kv_exp2(p[j][e] - mg[e & 1]);
                    sum[e & 1] += !none && vs[j] != vs[j] ? vs[j] : w;   // a NaN scale reaches the rows that see it
                    fx[(2 * t + (e & 1)) * 68 + 16 * j + g + 8 * (e >> 1)] = __float2uint_rn(w * ratio);
                }
            }
#pragma unroll
            for (int e = 0; e < 2; e++) {
                l[e] = l[e] * alpha[e] + wt[e] * sum[e];
                wt[e] *= vmax * (1.0f / DG::kP);
            }
            __syncwarp();
            uint32_t pd[D][4];   // row g, tokens 16 h + 4 t..+3 for h = 0..3
#pragma unroll
            for (int h = 0; h < 4; h++) {
                const uint4 f = *reinterpret_cast<const uint4*>(fx + g * 68 + 16 * h + 4 * t);
#pragma unroll
                for (int d = 0; d < D; d++) {
                    const int b = D - 1 - d, sel = b | (b + 4) << 4;
                    pd[d][h] = __byte_perm(__byte_perm(f.x, f.y, sel), __byte_perm(f.z, f.w, sel), 0x5410);
                }
            }
            __syncwarp();
            if (i + 1 < n) copy(i1, vp, vdst, slot);   // the next group's V into the slot of this group's K
            cp_async_commit();
            slot = slot == 2 ? 0 : slot + 1;
            // ---- out += V^T w
            cp_async_wait<2>();
            __syncwarp();
            const unsigned char* v8 = ring + slot * SM::kSlot;
#pragma unroll
            for (int w = 0; w < NW; w++) {
                const int seg = HDP == 128 ? (w ^ t) * 32 : (w ^ (t & 1)) * 32;
                uint32_t f[4][4];   // [16 tokens][dimension 32 w + 4 g + b]: tokens 16 h + 4 t..+3
#pragma unroll
                for (int h = 0; h < 4; h++) {
                    const unsigned char* at = v8 + (16 * h + 4 * t) * HDP + seg + 4 * g;
                    transpose4(*reinterpret_cast<const uint32_t*>(at), *reinterpret_cast<const uint32_t*>(at + HDP),
                               *reinterpret_cast<const uint32_t*>(at + 2 * HDP),
                               *reinterpret_cast<const uint32_t*>(at + 3 * HDP), f[h]);
                }
#pragma unroll
                for (int mt = 0; mt < 2; mt++) {
                    int acc[D][4];
                    const uint32_t f0[4] = {f[0][2 * mt], f[0][2 * mt + 1], f[1][2 * mt], f[1][2 * mt + 1]};
                    const uint32_t f1[4] = {f[2][2 * mt], f[2][2 * mt + 1], f[3][2 * mt], f[3][2 * mt + 1]};
#pragma unroll
                    for (int d = 0; d < D; d++) {
                        acc[d][0] = acc[d][1] = acc[d][2] = acc[d][3] = 0;
                        mma_su(acc[d], f0, pd[d][0], pd[d][1]);
                        mma_su(acc[d], f1, pd[d][2], pd[d][3]);
                    }
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        o[w][mt][e] = fmaf(DG::join(acc, e), wt[e & 1], o[w][mt][e] * alpha[e & 1]);
                }
            }
            __syncwarp();
            // ---- two groups on: its K into the slot of this group's V; three on: its pages
            if (i + 2 < n) {
                vet(i2);
                copy(i2, kp, kdst, slot);
                sc2 = scale_of(i2);
            }
            cp_async_commit();
            slot = slot == 2 ? 0 : slot + 1;
            if (i + 3 < n) {
                ahead.next(a);
                i3 = look(ahead);
            }
            i0 = i1;
            i1 = i2;
            i2 = i3;
            sc0 = sc1;
            sc1 = sc2;
        }
        cp_async_wait<0>();
        // what the warp holds of its last unit
        if (fresh && cur.g + 1 == cur.q.ng) put_rows();
        else put_piece(fresh ? reinterpret_cast<float*>(ring) : piece0, fresh, (int)(w1 - 1 - b0));
    }

    // ---- units that warps share, and what is left of them for other blocks
    KvPart* parts = a.whole ? nullptr : a.parts + 2 * (size_t)blockIdx.x;
    if (parts && threadIdx.x < 2) {
        parts[threadIdx.x].valid = 0;
        parts[threadIdx.x].at = b0;
    }
    __syncthreads();
    const int nblk = (int)(b1 - b0);
    for (int first = warp; first < 2 * kKvaWarps; first += kKvaWarps) {
        const typename SM::Info f = info[first];
        if (!f.valid) continue;
        int prev = first - 1;
        while (prev >= 0 && !info[prev].valid) prev--;
        if (prev >= 0 && info[prev].begin == f.begin) continue;   // the unit's first piece leads
        const bool all = f.begin >= 0 && f.end <= nblk;
        KvPart* part = all ? nullptr : parts + (f.begin <= 0 ? 0 : 1);
        if (!all && lane == 0) {
            part->begin = b0 + f.begin;
            part->end = b0 + f.end;
            part->s = f.s;
            part->h = f.h;
            part->rg = f.rg;
            part->valid = 1;
        }
        const KvSeq q = kv_seq(a, f.s);
        auto piece = [&](int i) {
            return reinterpret_cast<const float*>(
                i & 1 ? smem + (i >> 1) * SM::kRing : smem + kKvaWarps * SM::kRing + (i >> 1) * SM::kPiece);
        };
        for (int r = 0; r < kKvaRows; r++) {
            const KvRow row = kv_row(a, q, f.h, f.rg, r);
            if (row.out < 0) break;
            float mx = -INFINITY, ls = 0.0f, os[HDP / 32];
            for (int i = first; i < 2 * kKvaWarps; i++)
                if (info[i].valid && info[i].begin == f.begin) mx = fmaxf(mx, piece(i)[kKvaRows * HDP + r]);
#pragma unroll
            for (int e = 0; e < HDP / 32; e++) os[e] = 0.0f;
            for (int i = first; i < 2 * kKvaWarps; i++) {
                if (!info[i].valid || info[i].begin != f.begin) continue;
                const float* p = piece(i);
                const float pm = p[kKvaRows * HDP + r], wgt = pm == -INFINITY ? 0.0f : kv_exp2(pm - mx);
                ls += wgt * p[kKvaRows * HDP + kKvaRows + r];
#pragma unroll
                for (int e = 0; e < HDP / 32; e++) os[e] += wgt * p[r * HDP + (HDP / 32) * lane + e];
            }
            const int d0 = (HDP / 32) * lane;
            if (all) {
                const float inv = ls == 0.0f ? 0.0f : 1.0f / ls;
#pragma unroll
                for (int e = 0; e < HDP / 32; e++)
                    if (d0 + e < c.hd) ((T*)a.out)[row.out + d0 + e] = from_f32<T>(os[e] * inv);
            } else {
#pragma unroll
                for (int e = 0; e < HDP / 32; e++) part->o[r][d0 + e] = os[e];
                if (lane == 0) {
                    part->m[r] = mx;
                    part->l[r] = ls;
                }
            }
        }
    }
}

// Units that blocks share.  Block b - 1 takes the border before block b: the
// unit that lies across it, if this is the first border inside the unit.
constexpr int kKvJoinThreads = 128;
template <typename T>
__global__ void __launch_bounds__(kKvJoinThreads) k_kv_attention_join(const KvAttnArgs a, int blocks) {
    pdl_wait();
    const int b = blockIdx.x + 1, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const KvPart* lead = a.parts + 2 * (size_t)b;
    if (!lead->valid || lead->begin >= lead->at) return;
    const long long begin = lead->begin, before = a.parts[2 * (size_t)(b - 1)].at;
    if (begin < before) return;
    const KvPart* head = a.parts + 2 * (size_t)(b - 1) + (begin == before ? 0 : 1);
    int end = b + 1;
    while (end < blocks && a.parts[2 * (size_t)end].valid && a.parts[2 * (size_t)end].begin == begin) end++;
    const KvSeq q = kv_seq(a, lead->s);
    for (int r = warp; r < kKvaRows; r += kKvJoinThreads / 32) {
        const KvRow row = kv_row(a, q, lead->h, lead->rg, r);
        if (row.out < 0) break;
        float mx = head->m[r];
        for (int i = b; i < end; i++) mx = fmaxf(mx, a.parts[2 * (size_t)i].m[r]);
        float ls = 0.0f;
        float4 os = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int i = b - 1; i < end; i++) {
            const KvPart* p = i < b ? head : a.parts + 2 * (size_t)i;
            const float pm = p->m[r], wgt = pm == -INFINITY ? 0.0f : kv_exp2(pm - mx);
            const float4 x = *reinterpret_cast<const float4*>(&p->o[r][4 * lane]);
            ls += wgt * p->l[r];
            os.x += wgt * x.x;
            os.y += wgt * x.y;
            os.z += wgt * x.z;
            os.w += wgt * x.w;
        }
        const float inv = ls == 0.0f ? 0.0f : 1.0f / ls;
        if (4 * lane < a.c.hd)
            store4((T*)a.out + row.out + 4 * lane, a.vec_out, make_float4(os.x * inv, os.y * inv, os.z * inv, os.w * inv));
    }
}

}  // namespace aion
