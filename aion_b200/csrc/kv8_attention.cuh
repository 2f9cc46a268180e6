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
    int unit_log;                // rows of a unit of k_kv_attention: 1 << unit_log
    int whole;                   // blocks take whole units: nothing is left to join
    struct KvPart* parts;        // [blocks][2], else
};

// ---------------------------------------------------------------------------
// Arithmetic.  K and V stay the int8 values that the cache holds; the query
// becomes a fixed-point number of 3 base-256 digits and the softmax weights of
// D, so that every product is an exact integer dot on the tensor cores
// (mma.sync.m16n8k32, s32 accumulators):
//   q = rint(x 127 256^2 / max|x|), digits in -128..127, per row;
//   score = max|x| / (127 256^2) * K scale * sum_d 256^(2-d) (K . q_d);
//   w = rint(2^(score - m) r (256^D - 1)), digits in 0..255;
//   out += V * 2^(m - running m) / (256^D - 1) * sum_d ....
// V is the largest V scale of a group of 64 positions and r a position's own,
// relative to it; m is the group's largest score + log2 r that the row sees, so
// the largest 2^(score - m) r is 1, whatever the scales of pages that the row
// does not see, or hardly weighs (log2 r is cut off at -80, which bounds the sum
// of 2^(score - m)).
// A query's step is 2^-23 of its largest value, fp32's own, for 16-bit rows
// too: an error of a score is exponentiated, and with two digits (a step of
// 2^-15) an fp16 row with one channel 256 times the others lost scores of 0.01.
// D is 3 for fp32 rows and 2 for 16-bit rows, whose weights enter linearly: half
// a step, 2^-17 of the largest of 64, against the 2^-9 or 2^-12 of a rounded
// result.  Weights are relative to the largest of their group, so a position
// far below its row's maximum keeps its share.  Sums run in fp32.
//
// Rows and digits are the columns of the MMAs (8 of them).  WIDE: 8 rows, an
// MMA for each digit, which a lane joins by itself.  Else one MMA holds 4 rows
// x 2 digits (lane t of a quad has both of row t; a query's third digit has an
// MMA with every other column) or 2 rows x 3 digits in fours (two lanes have a
// row and swap halves), and half or less of the work around the MMAs is left:
// one query head per K/V head, or few, as most models decode.
//
// Work.  A unit is (sequence, K/V head, so many rows: tokens x query heads of
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
// pieces (cp.async), XOR-swizzled so that the eight rows that one phase of an
// ldmatrix reads lie in different banks.  K fragments (tokens x dimensions) are
// plain ldmatrix, V fragments (dimensions x tokens) its transposing 8-bit form.
// Page numbers and scales pass through shared memory, too: a register that
// waits for memory would hold up the warp when the pipeline moves on.  Loops
// over the head size run to its bound without branches (digits past it are
// zero): each branch keeps the MMAs around it from overlapping.
//
// Bound by memory where sequences are long: 16 x 8193..32767 bf16 tokens, 32
// query heads on 8, take 120 to 125 us (672 MB, 5.4 to 5.6 TB/s), one of 131072
// fp16 tokens 60 us (269 MB, 4.5 TB/s).  32 x 512..639 fp32 tokens of 32 heads
// take 37 us (153 MB) in a cache of at most 1024 tokens a sequence: there the
// start (the line, the first pages, the first rows: about 8 us) and the joins
// weigh, and a wider table adds the join's launch.  8 x 3..5 drafted fp32 rows
// of 40 heads on 251..1777 tokens take 41 us (85 MB), with 4 or 5 turns a warp.
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
// 16 rows x 32 bytes as an A fragment: lanes 0..15 give the rows' first 16
// bytes, lanes 16..31 their second.
__device__ __forceinline__ void ldsm_rows(uint32_t (&a)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3])
                 : "r"(addr)
                 : "memory");
}
// 32 rows x 16 bytes, transposed, as an A fragment of 16 x 32: lane i gives row i.
__device__ __forceinline__ void ldsm_cols(uint32_t (&a)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0,%1,%2,%3}, [%4];"
                 : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3])
                 : "r"(addr)
                 : "memory");
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
__device__ __forceinline__ void cp_async4(void* dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_addr(dst)), "l"(src) : "memory");
}

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
    q.nrg = (q.cnt * a.group + (1 << a.unit_log) - 1) >> a.unit_log;
    return q;
}

// Records what is wrong with a sequence: a slot that does not exist, positions behind its table.
__device__ __forceinline__ void kv_vet_seq(const KvAttnArgs& a, const KvSeq& q) {
    if (q.p0 < 0 || q.cnt == 0) return;
    if (q.slot < 0 || q.slot >= a.c.max_seqs) kv_flag(a.c, KV_BAD_ARG);
    else if ((long long)q.p0 + q.cnt > q.len) kv_flag(a.c, KV_BAD_PAGE);
}

// x / d for x >= 0, d > 0; 64-bit division is a long sequence, so it is kept for what needs it.
__device__ __forceinline__ long long kv_div(long long x, int d) {
    if ((x >> 32) == 0) return (uint32_t)x / (uint32_t)d;
    return x / d;
}

// A place in the line of groups.
struct KvCursor {
    KvSeq q;
    int s, h, rg, g;
    __device__ __forceinline__ void seek(const KvAttnArgs& a, int seq, long long rest) {
        s = seq;
        q = kv_seq(a, s);
        const long long u = kv_div(rest, q.ng);
        g = (int)(rest - u * q.ng);
        h = (int)kv_div(u, q.nrg);
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

// Rows of a unit as the lanes see them.
struct KvRow {
    long long q, out;   // element offsets; out -1: no row
    int lim;            // last position seen; -1: none
};
__device__ __forceinline__ KvRow kv_row(const KvAttnArgs& a, const KvSeq& q, int h, int rg, int r) {
    KvRow w;
    const int i = (rg << a.unit_log) + r, tok = i / a.group, head = h * a.group + (i - tok * a.group);
    const bool row = i < q.cnt * a.group;
    w.lim = row ? (int)min((long long)q.p0 + tok, (long long)q.len - 1) : -1;
    w.q = (q.t0 + tok) * a.q_stride + (long long)head * a.c.hd;
    w.out = row ? (q.t0 + tok) * a.out_stride + (long long)head * a.c.hd : -1;
    return w;
}

template <int HDP, int D, bool WIDE> struct KvaShape {
    static constexpr int kUnitLog = WIDE ? 3 : D == 2 ? 2 : 1, kUnit = 1 << kUnitLog;   // rows
    static constexpr int kSlot = kKvaT * HDP;
    static constexpr int kRing = 3 * kSlot;
    static constexpr int kPiece = (kUnit * HDP + 2 * kUnit) * 4;   // o, m, l
    static constexpr int kWords = D == 2 && !WIDE ? 36 : 68;   // of a row of weights: 64 of them (16-bit for 4 rows x 2 digits), padded
    static_assert(kRing % 16 == 0 && kUnit * kWords * 4 <= kSlot && kPiece <= kRing && kPiece % 16 == 0, "the places of the weights and pieces");
    struct Info {   // of a piece; the unit's groups from the block's first one on
        int begin, end, s, h, rg, rows;   // rows 0: no piece
    };
    static constexpr int kQueue = (4 * 4 + 4 * 8) * 4;   // pages and scales of four groups
    static constexpr int kPieces = kKvaWarps * kRing, kQueues = kPieces + kKvaWarps * kPiece;
    static constexpr int kInfo = kQueues + kKvaWarps * kQueue;
    static constexpr int kSums = kInfo + 2 * kKvaWarps * (int)sizeof(Info);   // warps' sums, the block's stretch
    static constexpr int kTotal = kSums + (kKvaWarps + 2) * 8;
    static_assert(kSums % 8 == 0 && kTotal <= 227 * 1024, "shared memory");
    static constexpr int kBlocks = 2 * (kTotal + 1024 + 128) <= 228 * 1024 ? 2 : 1;   // blocks an SM has room for
};

// The digits' dots of N accumulators, joined: values e < NV of a lane; `odd`: lane & 1.
__device__ __forceinline__ float kva_three(int a, int b, int c) {
    return fmaf((float)a, 65536.0f, fmaf((float)b, 256.0f, (float)c));
}
template <bool WIDE, int D, int N, int NV>
__device__ __forceinline__ void kva_join(const int (&acc)[N][4], bool odd, float (&v)[NV]) {
    if constexpr (WIDE) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if constexpr (N == 3) v[e] = kva_three(acc[0][e], acc[1][e], acc[2][e]);
            else v[e] = fmaf((float)acc[0][e], 256.0f, (float)acc[1][e]);
        }
    } else if constexpr (N == 2) {   // a query's digits 0 and 1 in one, 2 in the other
        v[0] = kva_three(acc[0][0], acc[0][1], acc[1][0]);
        v[1] = kva_three(acc[0][2], acc[0][3], acc[1][2]);
    } else if constexpr (D == 2) {
        v[0] = fmaf((float)acc[0][0], 256.0f, (float)acc[0][1]);
        v[1] = fmaf((float)acc[0][2], 256.0f, (float)acc[0][3]);
    } else {   // even lanes have digits 0 and 1, odd ones digit 2; even ones keep the first 8 of 16, odd ones the others
        const float lo = odd ? (float)acc[0][0] : fmaf((float)acc[0][0], 65536.0f, (float)acc[0][1] * 256.0f);
        const float hi = odd ? (float)acc[0][2] : fmaf((float)acc[0][2], 65536.0f, (float)acc[0][3] * 256.0f);
        v[0] = (odd ? hi : lo) + __shfl_xor_sync(0xffffffffu, odd ? lo : hi, 1);
    }
}

template <typename T, int HDP, int D, bool WIDE>
__global__ void __launch_bounds__(kKvaThreads, KvaShape<HDP, D, WIDE>::kBlocks) k_kv_attention(const KvAttnArgs a) {
    using SH = KvaShape<HDP, D, WIDE>;
    constexpr float kQ = 127.0f * 65536.0f, kP = D == 3 ? 16777215.0f : 65535.0f;
    constexpr float kUp = D == 3 ? 16777216.0f : 65536.0f;   // keeps the factor of a small V scale a normal number
    constexpr int KS = HDP / 32, MT = HDP / 16;   // k-steps of a score, 16-dimension tiles of a result
    constexpr int RL = WIDE ? 2 : 1;              // rows a lane has scores of
    constexpr int NV = WIDE ? 4 : D == 2 ? 2 : 1; // its scores of 16 positions
    constexpr int NQ = WIDE ? 3 : D == 2 ? 2 : 1; // MMAs for the digits of a query
    constexpr int ND = WIDE ? D : 1;              // and of the weights
    extern __shared__ __align__(16) unsigned char smem[];
    if (!a.whole) pdl_launch_dependents();   // the join's launch overlaps; it waits for this grid before it reads
    const KvView& c = a.c;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    unsigned char* ring = smem + warp * SH::kRing;
    float* piece0 = reinterpret_cast<float*>(smem + SH::kPieces + warp * SH::kPiece);
    int* q_page = reinterpret_cast<int*>(smem + SH::kQueues + warp * SH::kQueue);   // [4][4]: of the 16-key tiles of a group
    float* q_scale = reinterpret_cast<float*>(q_page + 16);                         // [4][8]: K scales, V scales
    typename SH::Info* info = reinterpret_cast<typename SH::Info*>(smem + SH::kInfo);
    long long *s_red = reinterpret_cast<long long*>(smem + SH::kSums), *s_range = s_red + kKvaWarps;

    if (blockIdx.x == 0) kv_vet_rows(c, a.r, threadIdx.x, kKvaThreads);
    // ---- the line: prefix sums of the sequences' groups (in the ring's memory), the block's and the warp's stretch
    long long* pre = reinterpret_cast<long long*>(smem);
    const int per = (a.r.n_seq + kKvaThreads - 1) / kKvaThreads, sa = min((int)threadIdx.x * per, a.r.n_seq),
              sb = min(sa + per, a.r.n_seq);
    long long mine = 0;
    for (int s = sa; s < sb; s++) {
        const KvSeq q = kv_seq(a, s);
        if (blockIdx.x == 0) kv_vet_seq(a, q);
        pre[s] = mine;
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
    long long W = 0, base = x - mine;
#pragma unroll
    for (int w = 0; w < kKvaWarps; w++) {
        if (w < warp) base += s_red[w];
        W += s_red[w];
    }
    for (int s = sa; s < sb; s++) pre[s] += base;
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
    const int nb = (int)min((long long)gridDim.x, (W + kKvaWarps - 1) / kKvaWarps);
    const long long share = kv_div(W, max(nb, 1)), more = W - share * nb;   // the first `more` blocks take one group more
    auto start = [&](int b) { return b >= nb ? W : share * b + min((long long)b, more); };
    long long b0 = start(blockIdx.x), b1 = start(blockIdx.x + 1);
    if (a.whole) {   // up to the next unit's start
        if (threadIdx.x < 2) {
            long long v = threadIdx.x ? b1 : b0;
            if (v < W) {
                const int s = find(v);
                const long long ng = kv_seq(a, s).ng, rest = v - pre[s];
                v = pre[s] + kv_div(rest + ng - 1, (int)ng) * ng;
            }
            s_range[threadIdx.x] = v;
        }
        __syncthreads();
        b0 = s_range[0];
        b1 = s_range[1];
    }
    const long long w0 = b0 + (b1 - b0) * warp / kKvaWarps, w1 = b0 + (b1 - b0) * (warp + 1) / kKvaWarps;
    const int n = (int)(w1 - w0);
    KvCursor ahead;   // the group whose pages are looked up next
    if (n > 0) {
        const int s = find(w0);
        ahead.seek(a, s, w0 - pre[s]);
    }
    if (lane < 2) info[2 * warp + lane].rows = 0;
    __syncthreads();   // the ring is free

    // ---- copies
    constexpr int NE = HDP / 32;   // a lane's pieces of 16 rows: source 16 (lane + 32 e)
    int dst[NE];
    const int cpr = c.hd / 16;
    auto place = [](int row, int ch) {
        return HDP == 128 ? row * 128 + ((ch ^ (row & 7)) << 4) : row * 64 + ((ch ^ ((row >> 1) & 3)) << 4);
    };
#pragma unroll
    for (int e = 0; e < NE; e++) dst[e] = place((lane + 32 * e) / cpr, (lane + 32 * e) % cpr);
    struct Item {   // a group of the line; g: its number in the unit, the sign bit says that it is the unit's last
        int s, h, rg, g;
    };
    // The next group's place; its pages (lane j < 4: of 16 keys; -2: past the keys) go to queue entry k.
    auto take = [&](int k) {
        Item it = {ahead.s, ahead.h, ahead.rg, ahead.g | (ahead.g + 1 == ahead.q.ng ? (int)0x80000000 : 0)};
        if (lane < 4) {
            const int pos = ahead.g * kKvaT + 16 * lane;
            int* to = q_page + 4 * k + lane;
            if (pos < ahead.q.len) cp_async4(to, c.tables + (size_t)ahead.q.slot * c.max_pages + (pos >> c.page_log));
            else *to = -2;
        }
        ahead.next(a);
        return it;
    };
    // Rows of a group to a slot; `with_scales`: K, with which the scales of both come.
    auto copy = [&](const Item& it, int k, const int8_t* pool, int slot, bool with_scales) {
        int page = q_page[4 * k + t];
        if (page < 0 || page >= c.n_pages) {   // pages that are missing are left out
            if (page != -2 && with_scales) kv_flag(c, KV_BAD_PAGE);
            page = -1;
        }
        const long long unit = (long long)page * c.nkv + it.h;
        if (with_scales && lane < 8) {
            float* to = q_scale + 8 * k + lane;
            if (page >= 0) cp_async4(to, (lane < 4 ? c.k_scale : c.v_scale) + (long long)a.layer * c.n_pages * c.nkv + unit);
            else *to = -1.0f;
        }
        const int row0 = (it.g & 0x7FFFFFFF) * kKvaT + 16 * t;
        const long long at = page < 0 ? -1 : (unit * c.page + (row0 & (c.page - 1))) * c.hd;
        const uint32_t to = smem_addr(ring + slot * SH::kSlot);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const long long from = __shfl_sync(0xffffffffu, at, j);
            const int8_t* src = pool + from + 16 * lane;
#pragma unroll
            for (int e = 0; e < NE; e++)
                if (from >= 0 && lane + 32 * e < c.hd)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + j * 16 * HDP + dst[e]),
                                 "l"(src + 512 * e)
                                 : "memory");
        }
    };
    const int8_t *kp = c.k + a.layer * c.plane(), *vp = c.v + a.layer * c.plane();

    // ---- state of the unit in use
    auto my_row = [&](int e) { return WIDE ? 2 * t + e : D == 2 ? t : t >> 1; };   // rows a lane has scores of
    float o[MT][NV], m[RL], l[RL], rs[RL];
    int lim[RL];
    uint32_t qd[NQ][KS][2];
    // Lane (g, t) brings column g of the score MMAs: a row, or a digit of one; dimensions 32 k + 4 t..+3 and + 16.
    auto begin_unit = [&](const Item& it) {
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
            for (int e = 0; e < NV; e++) o[i][e] = 0.0f;
        const KvSeq q = kv_seq(a, it.s);
        const KvRow row = kv_row(a, q, it.h, it.rg, WIDE ? g : D == 2 ? g >> 1 : g >> 2);
        float4 v[KS][2];
        float top = 0.0f;
        bool bad = false;
        const T* src = (const T*)a.q + row.q;
        const int end = row.lim >= 0 ? c.hd : 0;
        auto load = [&](auto vec) {
#pragma unroll
            for (int k = 0; k < KS; k++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const int d0 = 32 * k + 16 * i + 4 * t;
                    v[k][i] = d0 < end ? load4(src + d0, vec.value) : make_float4(0, 0, 0, 0);
                }
        };
        if (a.vec_q) load(std::true_type{});
        else load(std::false_type{});
        uint32_t high = 0;
#pragma unroll
        for (int k = 0; k < KS; k++) high = kv_top4(kv_top4(high, v[k][0]), v[k][1]);
        bad = high >= 0x7F800000u;
        top = __uint_as_float(high);
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        bad = (__ballot_sync(0xffffffffu, bad) >> (4 * g)) & 15;
        // rows of tiny values are scaled up first, so that the factor stays finite
        const float up = top < 8.6736174e-19f ? 1.8446744e19f : 1.0f;   // 2^-60, 2^64
        const float f = top > 0.0f && !bad ? kQ / (top * up) : 0.0f;
#pragma unroll
        for (int k = 0; k < KS; k++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const float* w = reinterpret_cast<const float*>(&v[k][i]);
                int dg[3][4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    int z = bad ? 0 : __float2int_rn(w[e] * up * f);
#pragma unroll
                    for (int d = 2; d >= 0; d--) {
                        dg[d][e] = (int8_t)z;
                        z = (z - dg[d][e]) >> 8;
                    }
                }
                uint32_t pk[3];
#pragma unroll
                for (int d = 0; d < 3; d++) pk[d] = pack4(dg[d][0], dg[d][1], dg[d][2], dg[d][3]);
                if constexpr (WIDE) {
#pragma unroll
                    for (int d = 0; d < 3; d++) qd[d % NQ][k][i] = pk[d];
                } else if constexpr (D == 2) {
                    qd[0][k][i] = g & 1 ? pk[1] : pk[0];
                    qd[NQ - 1][k][i] = g & 1 ? 0u : pk[2];
                } else {
                    qd[0][k][i] = (g & 3) == 0 ? pk[0] : (g & 3) == 1 ? pk[1] : (g & 3) == 2 ? pk[2] : 0u;
                }
            }
        const float r = bad ? __int_as_float(0x7FC00000) : top / kQ * a.scale;
#pragma unroll
        for (int e = 0; e < RL; e++) {
            const int from = 4 * (WIDE ? 2 * t + e : D == 2 ? 2 * t : 4 * (t >> 1));   // a lane of that row
            rs[e] = __shfl_sync(0xffffffffu, r, from);
            lim[e] = __shfl_sync(0xffffffffu, row.lim, from);
            m[e] = -INFINITY;
            l[e] = 0.0f;
        }
    };
    auto sub = [&](int e) { return g + 8 * (WIDE ? e >> 1 : D == 2 ? e : t & 1); };   // of 16 positions, or dimensions
    constexpr int kLow = !WIDE && D == 3 ? 1 : 4;   // lanes that share a row differ in these bits: 4, 8, 16 and, here, 1
    // What the warp has of a unit that ends, or goes on elsewhere, with group `at` (from the block's first on).
    auto end_unit = [&](const Item& it, bool whole_unit, float* piece, int which, int at) {
#pragma unroll
        for (int e = 0; e < RL; e++) {
            if (kLow == 1) l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
            l[e] += __shfl_xor_sync(0xffffffffu, l[e], 4);
            l[e] += __shfl_xor_sync(0xffffffffu, l[e], 8);
            l[e] += __shfl_xor_sync(0xffffffffu, l[e], 16);
        }
        const KvSeq q = kv_seq(a, it.s);
        if (whole_unit) {
#pragma unroll
            for (int e = 0; e < RL; e++) {
                const KvRow row = kv_row(a, q, it.h, it.rg, my_row(e));
                if (row.out < 0) continue;
                const float inv = l[e] == 0.0f ? 0.0f : 1.0f / l[e];
                T* to = (T*)a.out + row.out;
#pragma unroll
                for (int i = 0; i < MT; i++)
                    if (16 * i < c.hd)
#pragma unroll
                        for (int k = e; k < NV; k += RL) to[16 * i + sub(k)] = from_f32<T>(o[i][k] * inv);
            }
            return;
        }
#pragma unroll
        for (int e = 0; e < RL; e++) {
            float* row = piece + my_row(e) * HDP;
#pragma unroll
            for (int i = 0; i < MT; i++)
#pragma unroll
                for (int k = e; k < NV; k += RL) row[16 * i + sub(k)] = o[i][k];
            if (g == 0) {
                piece[SH::kUnit * HDP + my_row(e)] = m[e];
                piece[SH::kUnit * HDP + SH::kUnit + my_row(e)] = l[e];
            }
        }
        const int gg = it.g & 0x7FFFFFFF;
        if (lane == 0)
            info[2 * warp + which] = {at - gg, at - gg + q.ng, it.s, it.h, it.rg,
                                      min(SH::kUnit, q.cnt * a.group - it.rg * SH::kUnit)};
    };

    // ---- the stretch.  Turn i uses group i; it also fetches V of i + 1, K of i + 2 and the pages of i + 3, and the
    // turns before 0 do only that.
    if (n > 0) {
        Item i0, i1, i2, i3;
        i0 = i1 = i2 = i3 = Item{0, 0, 0, 0};
        bool begins = true, fresh = false;
        int kslot = 0;   // of K of group i (2 i mod 3); V of i lies in the next one
#pragma unroll 1
        for (int i = -3; i < n; i++) {
            const int vslot = kslot == 2 ? 0 : kslot + 1;
            float alpha[RL], wt[RL];
            uint32_t pd[ND][4];   // weights as B fragments: 16 h + 4 t..+3 for h = 0..3
            if (i >= 0) {
                if (begins) {
                    begin_unit(i0);
                    fresh = (i0.g & 0x7FFFFFFF) == 0;
                    begins = false;
                }
                // ---- scores
                cp_async_wait<2>();
                __syncwarp();
                const int key0 = (i0.g & 0x7FFFFFFF) * kKvaT;
                const float4 kscale = *reinterpret_cast<const float4*>(q_scale + 8 * (i & 3));
                const float4 vscale = *reinterpret_cast<const float4*>(q_scale + 8 * (i & 3) + 4);
                const float ksc[4] = {kscale.x, kscale.y, kscale.z, kscale.w}, vs[4] = {vscale.x, vscale.y, vscale.z, vscale.w};
                const uint32_t ks = smem_addr(ring + kslot * SH::kSlot);
                const float vmax = fmaxf(0.0f, fmaxf(fmaxf(vs[0], vs[1]), fmaxf(vs[2], vs[3])));   // without a NaN or a missing page
                float part[4] = {kP, kP, kP, kP}, lv[4] = {0.0f, 0.0f, 0.0f, 0.0f};   // r (256^D - 1), log2 r
                if (c.page < kKvaT) {
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        part[j] = vs[j] > 0.0f ? vs[j] / vmax : 0.0f;
                        lv[j] = fmaxf(__log2f(part[j]), -80.0f);
                        part[j] *= kP;
                    }
                }
                float p[4][NV], mg[RL];
#pragma unroll
                for (int e = 0; e < RL; e++) mg[e] = -INFINITY;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    int acc[NQ][4];
#pragma unroll
                    for (int d = 0; d < NQ; d++) acc[d][0] = acc[d][1] = acc[d][2] = acc[d][3] = 0;
#pragma unroll
                    for (int k = 0; k < KS; k++) {
                        uint32_t f[4];
                        ldsm_rows(f, ks + 16 * j * HDP + place(lane & 15, 2 * k + (lane >> 4)));
#pragma unroll
                        for (int d = 0; d < NQ; d++) mma_ss(acc[d], f, qd[d][k][0], qd[d][k][1]);
                    }
                    kva_join<WIDE, D>(acc, t & 1, p[j]);
#pragma unroll
                    for (int e = 0; e < NV; e++) {
                        const int pos = ksc[j] == -1.0f ? 0x7FFFFFFF : key0 + 16 * j + sub(e);   // -1: no page
                        p[j][e] = pos <= lim[e % RL] ? p[j][e] * (rs[e % RL] * ksc[j]) : -INFINITY;
                        mg[e % RL] = fmaxf(mg[e % RL], p[j][e] + lv[j]);
                    }
                }
                // ---- weights relative to the group's largest
#pragma unroll
                for (int e = 0; e < RL; e++) {
                    if (kLow == 1) mg[e] = fmaxf(mg[e], __shfl_xor_sync(0xffffffffu, mg[e], 1));
                    mg[e] = fmaxf(mg[e], __shfl_xor_sync(0xffffffffu, mg[e], 4));
                    mg[e] = fmaxf(mg[e], __shfl_xor_sync(0xffffffffu, mg[e], 8));
                    mg[e] = fmaxf(mg[e], __shfl_xor_sync(0xffffffffu, mg[e], 16));
                    const float mn = fmaxf(m[e], mg[e]);
                    alpha[e] = m[e] == -INFINITY ? 0.0f : kv_exp2(m[e] - mn);
                    wt[e] = mg[e] == -INFINITY ? 0.0f : kv_exp2(mg[e] - mn);
                    m[e] = mn;
                    if (mg[e] == -INFINITY) mg[e] = 0.0f;   // nothing seen: weights of 2^-inf
                }
                uint32_t* fx = reinterpret_cast<uint32_t*>(ring + kslot * SH::kSlot);   // K is read: [row][kWords]
                __syncwarp();
                float sum[RL] = {};
#pragma unroll
                for (int j = 0; j < 4; j++) {
#pragma unroll
                    for (int e = 0; e < NV; e++) {
                        const float w = kv_exp2(p[j][e] - mg[e % RL]);
                        sum[e % RL] += w;
                        if (vs[j] != vs[j] && p[j][e] != -INFINITY) sum[e % RL] = vs[j];   // a NaN scale reaches the rows that see it
                        const uint32_t z = __float2uint_rn(fminf(w * part[j], kP));   // lv is rounded
                        const int at = 16 * j + sub(e);
                        if constexpr (D == 2 && !WIDE) reinterpret_cast<uint16_t*>(fx + my_row(0) * SH::kWords)[at] = (uint16_t)z;
                        else fx[my_row(e % RL) * SH::kWords + at] = z;
                    }
                }
#pragma unroll
                for (int e = 0; e < RL; e++) {
                    l[e] = l[e] * alpha[e] + wt[e] * sum[e];
                    wt[e] *= vmax * (kUp / kP);
                }
                __syncwarp();
#pragma unroll
                for (int h = 0; h < 4; h++) {
                    if constexpr (D == 2 && !WIDE) {   // column g: row g >> 1, digit g & 1
                        const uint2 f = *reinterpret_cast<const uint2*>(fx + (g >> 1) * SH::kWords + 8 * h + 2 * t);
                        pd[0][h] = __byte_perm(f.x, f.y, g & 1 ? 0x6420 : 0x7531);
                    } else {
                        const uint4 f = *reinterpret_cast<const uint4*>(fx + (WIDE ? g : g >> 2) * SH::kWords + 16 * h + 4 * t);
#pragma unroll
                        for (int d = 0; d < ND; d++) {
                            const int b = WIDE ? D - 1 - d : 2 - min(g & 3, 2), sel = b | (b + 4) << 4;
                            pd[d][h] = __byte_perm(__byte_perm(f.x, f.y, sel), __byte_perm(f.z, f.w, sel), 0x5410);
                        }
                        if (!WIDE && (g & 3) == 3) pd[0][h] = 0;
                    }
                }
                __syncwarp();
            }
            if (i + 3 < n) i3 = take((i + 3) & 3);
            if (i >= -1 && i + 1 < n) copy(i1, (i + 1) & 3, vp, kslot, false);   // over K of group i
            cp_async_commit();
            if (i >= 0) {
                // ---- out += V^T w
                cp_async_wait<2>();
                __syncwarp();
                const uint32_t v8 = smem_addr(ring + vslot * SH::kSlot);
#pragma unroll
                for (int mt = 0; mt < MT; mt++) {
                    int acc[ND][4];
#pragma unroll
                    for (int d = 0; d < ND; d++) acc[d][0] = acc[d][1] = acc[d][2] = acc[d][3] = 0;
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        uint32_t f[4];
                        ldsm_cols(f, v8 + 32 * k * HDP + place(lane, mt));
#pragma unroll
                        for (int d = 0; d < ND; d++) mma_su(acc[d], f, pd[d][2 * k], pd[d][2 * k + 1]);
                    }
                    float v[NV];
                    kva_join<WIDE, D>(acc, t & 1, v);
#pragma unroll
                    for (int e = 0; e < NV; e++) o[mt][e] = fmaf(v[e] * (1.0f / kUp), wt[e % RL], o[mt][e] * alpha[e % RL]);
                }
                __syncwarp();
                if (i0.g < 0 || i + 1 == n) {   // the unit's last group, or the stretch's
                    const bool all = i0.g < 0 && fresh;
                    end_unit(i0, all, fresh ? reinterpret_cast<float*>(ring) : piece0, fresh, (int)(w0 - b0) + i);
                    begins = true;
                }
            }
            if (i >= -2 && i + 2 < n) {   // over V of group i; its pages are there, as the last wait says
                if (i == -2) {   // pages of groups 0 and 1: those of 2 on are there by the waits of the turns
                    cp_async_wait<0>();
                    __syncwarp();
                }
                copy(i2, (i + 2) & 3, kp, vslot, true);
            }
            cp_async_commit();
            kslot = vslot == 2 ? 0 : vslot + 1;
            i0 = i1;
            i1 = i2;
            i2 = i3;
        }
    }

    // ---- units that warps share, and what is left of them for other blocks
    KvPart* parts = a.whole ? nullptr : a.parts + 2 * (size_t)blockIdx.x;
    if (parts && threadIdx.x < 2) {
        parts[threadIdx.x].valid = 0;
        parts[threadIdx.x].at = b0;
    }
    __syncthreads();
    // Pieces in the line's order are 0..15 (a warp's first and last); the first piece of each unit leads.  Warps take
    // (unit, row) in turn: lane i weighs piece i.
    const int nblk = (int)(b1 - b0);
    const typename SH::Info mine_info = info[lane & 15];
    const unsigned have = __ballot_sync(0xffffffffu, lane < 16 && mine_info.rows);
    int task = 0;
#pragma unroll 1
    for (unsigned todo = have; todo;) {
        const int lead = __ffs(todo) - 1;
        const int begin = __shfl_sync(0xffffffffu, mine_info.begin, lead), end = __shfl_sync(0xffffffffu, mine_info.end, lead);
        const unsigned group = __ballot_sync(0xffffffffu, lane < 16 && mine_info.rows && mine_info.begin == begin);
        todo &= ~group;
        const int us = __shfl_sync(0xffffffffu, mine_info.s, lead), uh = __shfl_sync(0xffffffffu, mine_info.h, lead),
                  urg = __shfl_sync(0xffffffffu, mine_info.rg, lead);
        const bool all = begin >= 0 && end <= nblk;
        KvPart* part = all ? nullptr : parts + (begin <= 0 ? 0 : 1);
        if (!all && threadIdx.x == 0) {
            part->begin = b0 + begin;
            part->end = b0 + end;
            part->s = us;
            part->h = uh;
            part->rg = urg;
            part->valid = 1;
        }
        const int rows = __shfl_sync(0xffffffffu, mine_info.rows, lead);
        const float* piece = reinterpret_cast<const float*>(lane & 1 ? smem + ((lane >> 1) & 7) * SH::kRing
                                                                     : smem + SH::kPieces + ((lane >> 1) & 7) * SH::kPiece);
#pragma unroll 1
        for (int r = 0; r < rows; r++, task++) {
            if ((task & (kKvaWarps - 1)) != warp) continue;
            const bool in = (group >> lane) & 1;
            const float pm = in ? piece[SH::kUnit * HDP + r] : -INFINITY;
            const float mx = warp_max(pm), wgt = pm == -INFINITY ? 0.0f : kv_exp2(pm - mx);
            const float ls = warp_sum(in ? wgt * piece[SH::kUnit * HDP + SH::kUnit + r] : 0.0f);
            float os[HDP / 32] = {};
#pragma unroll 4
            for (int i = 0; i < 16; i++) {
                const float w = __shfl_sync(0xffffffffu, wgt, i);
                if (!((group >> i) & 1)) continue;
                const float* p = reinterpret_cast<const float*>(i & 1 ? smem + (i >> 1) * SH::kRing
                                                                      : smem + SH::kPieces + (i >> 1) * SH::kPiece);
#pragma unroll
                for (int e = 0; e < HDP / 32; e++) os[e] += w * p[r * HDP + lane + 32 * e];
            }
            if (all) {
                const KvRow row = kv_row(a, kv_seq(a, us), uh, urg, r);
                const float inv = ls == 0.0f ? 0.0f : 1.0f / ls;
#pragma unroll
                for (int e = 0; e < HDP / 32; e++)
                    if (lane + 32 * e < c.hd) ((T*)a.out)[row.out + lane + 32 * e] = from_f32<T>(os[e] * inv);
            } else {
#pragma unroll
                for (int e = 0; e < HDP / 32; e++) part->o[r][lane + 32 * e] = os[e];
                if (lane == 0) {
                    part->m[r] = mx;
                    part->l[r] = ls;
                }
            }
        }
    }
}

// Units that blocks share.  Block b - 1 takes the border before block b: the
// unit that lies across it, if this is the first border inside the unit.  The
// records of the blocks from b - 1 on are read at once, lane i that of b - 1 + i.
constexpr int kKvJoinThreads = 256;   // a warp a row: one trip after the other is what this costs
template <typename T>
__global__ void __launch_bounds__(kKvJoinThreads) k_kv_attention_join(const KvAttnArgs a, int blocks) {
    static_assert(kKvJoinThreads / 32 >= kKvaRows, "a warp for each row");
    const int b = blockIdx.x + 1, r = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (r >= 1 << a.unit_log) return;
    pdl_wait();
    const KvPart* p0 = a.parts + 2 * (size_t)(b - 1);
    const KvPart* mine = p0 + 2 * (size_t)lane;
    const bool there = b - 1 + lane < blocks;
    const long long begin = there && mine->valid ? mine->begin : -1, at = there ? mine->at : -1;
    const KvPart* lead = p0 + 2;
    const int s = lead->s, h = lead->h, rg = lead->rg;
    const long long ubegin = __shfl_sync(0xffffffffu, begin, 1), uat = __shfl_sync(0xffffffffu, at, 1);
    const long long before = __shfl_sync(0xffffffffu, at, 0);
    if (ubegin < 0 || ubegin >= uat || ubegin < before) return;
    const KvPart* head = p0 + (ubegin == before ? 0 : 1);
    // blocks b..end-1 hold a part in their first record; a unit over more than 31 blocks is followed one by one
    const unsigned other = ~__ballot_sync(0xffffffffu, lane == 0 || begin == ubegin);
    int end = b - 1 + (other ? __ffs(other) - 1 : 32);
    if (!other)
        while (end < blocks && a.parts[2 * (size_t)end].valid && a.parts[2 * (size_t)end].begin == ubegin) end++;
    const int np = end - (b - 1);
    const KvRow row = kv_row(a, kv_seq(a, s), h, rg, r);
    float mx = -INFINITY, ls = 0.0f;
    float4 os = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    // the parts of a row that the unit does not have are not set: it is joined all the same, and not stored
    for (int base = 0; base < np; base += 32) {   // lane i weighs part base + i
        const KvPart* p = base + lane == 0 ? head : p0 + 2 * (size_t)(base + lane);
        const bool in = base + lane < np;
        const float pm = in ? p->m[r] : -INFINITY, pl = in ? p->l[r] : 0.0f;
        const float mn = fmaxf(mx, warp_max(pm)), wgt = pm == -INFINITY ? 0.0f : kv_exp2(pm - mn);
        const float old = mx == -INFINITY ? 0.0f : kv_exp2(mx - mn);
        mx = mn;
        ls = ls * old + warp_sum(wgt * pl);
        os = make_float4(os.x * old, os.y * old, os.z * old, os.w * old);
        const int n = min(np - base, 32);
#pragma unroll 8
        for (int i = 0; i < n; i++) {
            const KvPart* pi = base + i == 0 ? head : p0 + 2 * (size_t)(base + i);
            const float w = __shfl_sync(0xffffffffu, wgt, i);
            const float4 x = *reinterpret_cast<const float4*>(&pi->o[r][4 * lane]);
            os.x += w * x.x;
            os.y += w * x.y;
            os.z += w * x.z;
            os.w += w * x.w;
        }
    }
    const float inv = ls == 0.0f ? 0.0f : 1.0f / ls;
    if (row.out >= 0 && 4 * lane < a.c.hd)
        store4((T*)a.out + row.out + 4 * lane, a.vec_out, make_float4(os.x * inv, os.y * inv, os.z * inv, os.w * inv));
}

}  // namespace aion
