// Attention over the 8-bit paged K/V cache (kv8.cuh) for many query rows a
// sequence: prompts and chunks of prompts, on the 5th-generation tensor cores.
#pragma once

#include "kv8_attention.cuh"
#include "tcgen05.cuh"

namespace aion {

// ---------------------------------------------------------------------------
// A block takes one K/V head and 256 rows (two tiles of 128) of a sequence: the
// rows of a K/V head are its tokens times the query heads that read it, so
// grouped heads share every key.  Keys come in tiles of 64:
//   warps 0-3, 4-7   softmax of row tile 0, 1: one thread a row;
//   warps 8-15       fetch K (warps 8, 9, 12, 13) and V (the others) with
//                    cp.async and bring them from int8 to fp16, which holds
//                    each value exactly, in 128-byte-swizzled shared memory,
//                    V transposed (tokens contiguous);
//   warps 16, 17     issue tcgen05.mma (kind::f16, M 128) for row tile 0, 1:
//                    S = Q K^T, then O += P V with P read from TMEM.
// Each role is a chain of waits, so none is given two tiles' or two operands'
// work; the softmax, the longest, takes registers from the others (setmaxnreg).
// Loops are kept short, and K and V warps on sub-partitions of their own: the
// roles of a sub-partition share its instruction cache.
// TMEM, for each row tile: two S buffers of 64 columns, O of 128.  P takes the
// place of its own S (which the softmax holds in registers by then), so S of
// key tile i + 2 waits for the MMAs that read P of tile i (pv_done: nothing
// else orders two MMAs of different accumulators), while the softmax works on
// tile i + 1.
//
// Arithmetic.  fp16 queries are taken as they are; bf16 and fp32 ones are
// scaled by a power of two per row so that the largest is below 2^15 (a bf16
// value then is an fp16 value, but for parts 2^-39 of the largest), and fp32
// ones are split into two fp16 terms (22 bits), each with its own MMA.
// Products of fp16 values are exact in the MMA and summed in fp32.
// P = 2^(s - m) * 2^7 * vscale / vref in fp16 (fp32 rows: two terms, 22
// bits; 16-bit rows: one, off by 2^-11 of itself at most, which is half a step
// of an fp16 result and an eighth of one of bf16), where vref is the largest V scale of the sequence's pages for this
// head, so that pages of different scales add up in one accumulator; the sum
// l of 2^(s - m) is kept in fp32 from the unrounded weights.  m is a running
// reference of s + log2(vscale / vref) over what the row sees, so that the
// largest P of a row is 2^7 or more whatever the scales of pages that it does
// not see, or hardly weighs.  (At -80 the logarithm is cut off, which bounds l
// by 2^88 a key: only pages that much below another lose bits.)  m follows
// the row's maximum only when that has grown by more than 8 (a factor of 2^8,
// and P stays below 2^15), which leaves O untouched for most tiles.
//
// A block of 256 rows takes 5K clocks to set up, 13K to bring fp32 queries in,
// 2.6K (16-bit rows) or 3.3K (fp32) a key tile and 7K to write; the MMAs alone
// would take 1.3K and 2.6K a tile.  2 x 1999..2048 bf16 rows of 32 heads on 8
// behind 4096..6143 tokens: 588 us, 0.41 TFLOP, 690 TFLOP/s, bound by the
// softmax and the 3.5 blocks an SM.  8 x 512 fp32 rows of 32 heads: 110 us,
// bound by what surrounds 2 to 8 key tiles of a block (its form spills 28 bytes
// a thread around the loop).
// ---------------------------------------------------------------------------
constexpr int kKvpThreads = 640, kKvpTile = 64;
constexpr int kKvpQ = 128 * 128 * 2;        // a query operand: 128 rows of two 128-byte-wide halves
constexpr int kKvpStage = 64 * 128 * 2;     // a key tile's K (64 rows, two halves) or V (up to 128 dimensions x 64 tokens)
constexpr int kKvpRaw = 64 * 128;           // a key tile's K or V as the cache holds it
constexpr int kKvpSmem = 2 * kKvpQ + 8 * kKvpStage + 4 * kKvpRaw + 1024;
constexpr uint32_t kKvpWaitLimit = 20000;
constexpr float kKvpLvMin = -80.0f;

// Registers a thread, by warpgroup; at launch all have 96 (640 threads).
constexpr int kKvpRegsSoft = 144, kKvpRegsConv = 72, kKvpRegsMma = 40;
static_assert(2 * kKvpRegsSoft + 2 * kKvpRegsConv + kKvpRegsMma <= 5 * 96, "the registers of the launch");
template <int N> __device__ __forceinline__ void regs_more() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void regs_less() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

__device__ __forceinline__ uint32_t kvp_idesc(int n) {   // fp16 A and B (K-major), fp32 D, M 128
    return (1u << 4) | ((uint32_t)(n >> 3) << 17) | (8u << 24);
}
// Loads and their wait are one instruction to the compiler: a register that a
// load is still on its way to cannot be moved or spilled.
__device__ __forceinline__ void tmem_ld64(uint32_t taddr, uint32_t (&x)[2][32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%64];\n\t"
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,"
        "%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%65];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(x[0][0]), "=r"(x[0][1]), "=r"(x[0][2]), "=r"(x[0][3]), "=r"(x[0][4]), "=r"(x[0][5]), "=r"(x[0][6]),
          "=r"(x[0][7]), "=r"(x[0][8]), "=r"(x[0][9]), "=r"(x[0][10]), "=r"(x[0][11]), "=r"(x[0][12]),
          "=r"(x[0][13]), "=r"(x[0][14]), "=r"(x[0][15]), "=r"(x[0][16]), "=r"(x[0][17]), "=r"(x[0][18]),
          "=r"(x[0][19]), "=r"(x[0][20]), "=r"(x[0][21]), "=r"(x[0][22]), "=r"(x[0][23]), "=r"(x[0][24]),
          "=r"(x[0][25]), "=r"(x[0][26]), "=r"(x[0][27]), "=r"(x[0][28]), "=r"(x[0][29]), "=r"(x[0][30]),
          "=r"(x[0][31]), "=r"(x[1][0]), "=r"(x[1][1]), "=r"(x[1][2]), "=r"(x[1][3]), "=r"(x[1][4]),
          "=r"(x[1][5]), "=r"(x[1][6]), "=r"(x[1][7]), "=r"(x[1][8]), "=r"(x[1][9]), "=r"(x[1][10]),
          "=r"(x[1][11]), "=r"(x[1][12]), "=r"(x[1][13]), "=r"(x[1][14]), "=r"(x[1][15]), "=r"(x[1][16]),
          "=r"(x[1][17]), "=r"(x[1][18]), "=r"(x[1][19]), "=r"(x[1][20]), "=r"(x[1][21]), "=r"(x[1][22]),
          "=r"(x[1][23]), "=r"(x[1][24]), "=r"(x[1][25]), "=r"(x[1][26]), "=r"(x[1][27]), "=r"(x[1][28]),
          "=r"(x[1][29]), "=r"(x[1][30]), "=r"(x[1][31])
        : "r"(taddr), "r"(taddr + 32)
        : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_smem_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ uint32_t half2_bits(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// Four int8 values of a word as two fp16 pairs: 1024 + (value + 128) is the
// fp16 pattern 0x6400 | (value ^ 0x80), and taking 1152 away is exact.
__device__ __forceinline__ uint2 int8x4_to_half(uint32_t w) {
    const uint32_t u = w ^ 0x80808080u, magic = 0x64646464u, off = 0x64806480u;
    uint32_t a = __byte_perm(u, magic, 0x4140), b = __byte_perm(u, magic, 0x4342);
    const __half2 o = *reinterpret_cast<const __half2*>(&off);
    const __half2 x = __hsub2(*reinterpret_cast<__half2*>(&a), o), y = __hsub2(*reinterpret_cast<__half2*>(&b), o);
    return make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
}
// Byte offset of 16-byte piece ch (8 values) of a row of an operand of `rows`
// rows, in halves of 64 values with the 128-byte swizzle.
__device__ __forceinline__ int kvp_piece(int rows, int row, int ch) {
    return (ch >> 3) * rows * 128 + row * 128 + (((ch & 7) ^ (row & 7)) << 4);
}

// Wait that gives up when the block has failed or after about two seconds.  A
// poll sleeps for up to 100 us, so that waiting warps leave the issue slots and
// the shared-memory pipe to the others.
__device__ __forceinline__ bool kvp_wait(uint64_t* bar, uint32_t parity, volatile int* fail) {
    const uint32_t b = smem_addr(bar);
    for (uint32_t i = 0; i < kKvpWaitLimit; i++) {
        uint32_t done;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, 100000;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(done)
            : "r"(b), "r"(parity)
            : "memory");
        if (done) return true;
        if (*fail) return false;
    }
    *fail = 1;
    return false;
}

// What the softmax needs to know of a key tile: for each 16 of its keys the
// scales, and which of them have a page.
struct alignas(16) KvpMeta {
    float ks[4], fv[4];   // fv = 2^7 vscale / vref; ks is not negative (1 where it is NaN or there is no page)
    float lv[4];          // log2(vscale / vref), kKvpLvMin at least
    uint32_t live, nan;   // bit j: keys 16 j.. have a page; one of its scales is NaN
};

template <typename T>
__global__ void __launch_bounds__(kKvpThreads, 1) k_kv_prompt(const KvAttnArgs a) {
    constexpr int TERMS = sizeof(T) == 4 ? 2 : 1;   // fp16 terms of a query and of a weight
    constexpr int NQ = 2, ROWS = 128 * NQ;
    constexpr int ST = TERMS == 2 ? 2 : 4;          // stages of K and of V
    static_assert(NQ * TERMS * kKvpQ + 2 * ST * kKvpStage + 4 * kKvpRaw + 1024 == kKvpSmem, "shared memory");
    extern __shared__ __align__(1024) unsigned char psm_raw[];
    __shared__ __align__(8) uint64_t q_full, k_full[ST], k_empty[ST], v_full[ST], v_empty[ST], s_full[NQ][2], p_full[NQ][2],
        pv_done[NQ], o_full[NQ], done_bar;
    __shared__ uint32_t s_tmem;
    __shared__ float s_red[4];
    __shared__ KvpMeta s_meta[8];
    __shared__ float s_scale[2][8];   // K and V scales of a tile's four pieces on their way; K scale -1: no page
    __shared__ volatile int s_fail;
    unsigned char* sm = psm_raw + ((1024u - (smem_addr(psm_raw) & 1023u)) & 1023u);
    unsigned char *qs = sm, *kst = sm + NQ * TERMS * kKvpQ, *vst = kst + ST * kKvpStage, *raw = vst + ST * kKvpStage;
    const KvView& c = a.c;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    // ---- the block's rows
    const int h = blockIdx.x % c.nkv, place = (gridDim.x - 1 - blockIdx.x) / c.nkv;   // late rows, which see most, first, in all heads
    int blk = 0, s = 0;
    {
        // places of a sequence: (rows before it / ROWS) + its number, on
        auto first = [&](int i) { return (int)((long long)a.r.begin(i) * a.group / ROWS) + i; };
        const int lo = kv_warp_find(a.r.n_seq, place, first);
        s = lo;
        blk = place - first(lo);
    }
    const KvSeq q = kv_seq(a, s);
    const long long total = (long long)q.cnt * a.group;
    if (blk < 0 || (long long)blk * ROWS >= total) {
        if (blockIdx.x == 0) kv_vet_rows(c, a.r, threadIdx.x, kKvpThreads);
        return;
    }
    const int row0 = blk * ROWS;
    const int rows = (int)min((long long)ROWS, total - row0);
    const int nq = rows > 128 ? 2 : 1;
    int nt[NQ];   // key tiles of each row tile: up to its last row's position
#pragma unroll
    for (int i = 0; i < NQ; i++) {
        const int last = min(row0 + 128 * (i + 1), row0 + rows) - 1;
        const long long seen = min((long long)q.p0 + last / a.group, (long long)q.len - 1) + 1;
        nt[i] = i < nq && q.len ? (int)((seen + kKvpTile - 1) / kKvpTile) : 0;
    }
    const int ntiles = nt[nq - 1];

    if (warp < 8) {   // the query rows to L2 while the block is set up
        const int i = row0 + 32 * warp + lane, tok = i / a.group;
        if (i < row0 + rows) {
            const T* src = (const T*)a.q + (q.t0 + tok) * a.q_stride + (long long)(h * a.group + i - tok * a.group) * c.hd;
            for (int d = 0; d < c.hd; d += 128 / (int)sizeof(T)) asm volatile("prefetch.global.L2 [%0];" ::"l"(src + d));
        }
    }
    if (threadIdx.x == 0) {
        kv_vet_seq(a, q);
        mbar_init(smem_addr(&q_full), 4 * NQ);
        for (int i = 0; i < ST; i++) {
            mbar_init(smem_addr(&k_full[i]), 4);
            mbar_init(smem_addr(&k_empty[i]), NQ);
            mbar_init(smem_addr(&v_full[i]), 4);
            mbar_init(smem_addr(&v_empty[i]), NQ);
        }
        for (int i = 0; i < NQ; i++) {
            for (int b = 0; b < 2; b++) {
                mbar_init(smem_addr(&s_full[i][b]), 1);
                mbar_init(smem_addr(&p_full[i][b]), 4);
            }
            mbar_init(smem_addr(&pv_done[i]), 1);
            mbar_init(smem_addr(&o_full[i]), 1);
        }
        mbar_init(smem_addr(&done_bar), NQ);
        s_fail = 0;
        fence_mbar_init();
    }
    if (warp == 16) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&s_tmem)), "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // ---- the largest V scale of the pages in sight
    float vref = 0.0f;
    const int32_t* table = c.tables + (size_t)(q.len ? q.slot : 0) * c.max_pages;
    if (warp >= 8 && warp < 12) {
        const int used = (int)(((long long)ntiles * kKvpTile < q.len ? (long long)ntiles * kKvpTile : q.len) + c.page - 1) >>
                         c.page_log;
        for (int i = threadIdx.x - 256; i < used; i += 128) {
            const int page = table[i];
            if (page >= 0 && page < c.n_pages)
                vref = fmaxf(vref, c.v_scale[((long long)a.layer * c.n_pages + page) * c.nkv + h]);   // without a NaN
        }
        vref = warp_max(vref);
        if (lane == 0) s_red[warp - 8] = vref;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    vref = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));

    if (warp < 8) {
        // ================= softmax: thread = row =================
        regs_more<kKvpRegsSoft>();
        const int tile = warp >> 2, r = threadIdx.x & 127, i = row0 + 128 * tile + r;
        const int tok = i / a.group, head = h * a.group + (i - tok * a.group);
        const bool live_row = i < total && 128 * tile + r < rows;
        const int lim = live_row ? (int)min((long long)q.p0 + tok, (long long)q.len - 1) : -1;
        // The warp's 32 query rows to shared memory, a row at a time so that its loads are one line after the other; lane l
        // has dimensions 4 l..+3, and keeps what row l's scores are scaled by.
        float rs = 1.0f;
        bool bad = false;
        {
            const long long mine = live_row ? (q.t0 + tok) * a.q_stride + (long long)head * c.hd : -1;
            const float sign = a.scale < 0.0f ? -1.0f : 1.0f;
            const bool in = 4 * lane < c.hd;
            // Lanes past the head size bring zeros, which no MMA reads.
            auto load = [&](int r0, float4 (&v)[4], auto vec) {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const long long from = __shfl_sync(0xffffffffu, mine, r0 + e);
                    v[e] = from >= 0 && in ? load4((const T*)a.q + from + 4 * lane, vec.value) : make_float4(0, 0, 0, 0);
                }
            };
            unsigned char* to0 = qs + tile * TERMS * kKvpQ + kvp_piece(128, 32 * (warp & 3), lane >> 1) + 8 * (lane & 1);
            auto put = [&](int r0, const float4 (&v)[4]) {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const uint32_t top = __reduce_max_sync(0xffffffffu, kv_top4(0, v[e]));
                    const bool off = top >= 0x7F800000u;
                    float up = 1.0f;   // the largest to 2^14..2^15, as far as a factor of 2^126 goes
                    if (!std::is_same<T, __half>::value && top != 0 && !off)
                        up = __uint_as_float((uint32_t)(127 + min(14 + 127 - (int)(top >> 23), 126)) << 23);
                    const float f = up * sign;
                    const float x0 = off ? 0.0f : v[e].x * f, x1 = off ? 0.0f : v[e].y * f, x2 = off ? 0.0f : v[e].z * f,
                                x3 = off ? 0.0f : v[e].w * f;
                    const uint2 hi = make_uint2(half2_bits(x0, x1), half2_bits(x2, x3));
                    // row r's pieces are swizzled with r & 7, which to0 has for row 0
                    const int row = r0 + e;
                    unsigned char* to = reinterpret_cast<unsigned char*>(reinterpret_cast<uintptr_t>(to0) ^ ((row & 7) << 4)) + row * 128;
                    *reinterpret_cast<uint2*>(to) = hi;
                    if (TERMS == 2) {
                        const float2 a0 = __half22float2(*reinterpret_cast<const __half2*>(&hi.x)),
                                     a1 = __half22float2(*reinterpret_cast<const __half2*>(&hi.y));
                        *reinterpret_cast<uint2*>(to + kKvpQ) =
                            make_uint2(half2_bits(x0 - a0.x, x1 - a0.y), half2_bits(x2 - a1.x, x3 - a1.y));
                    }
                    if (lane == row) {
                        rs = off ? 1.0f : fabsf(a.scale) / up;
                        bad = off;
                    }
                }
            };
            auto bring = [&](auto vec) {
                float4 va[4], vb[4];
                load(0, va, vec);
#pragma unroll 1
                for (int r0 = 0; r0 < 32; r0 += 8) {
                    load(r0 + 4, vb, vec);
                    put(r0, va);
                    load(min(r0 + 8, 28), va, vec);
                    put(r0 + 4, vb);
                }
            };
            if (a.vec_q) bring(std::true_type{});
            else bring(std::false_type{});
        }
        fence_smem_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_addr(&q_full));

        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
        const uint32_t to = tmem + lanes + 256 + 128 * tile;   // O
        float m = -INFINITY, l = 0.0f;   // a NaN in l stays and reaches the result
        const int mine = nt[tile];
        bool ok = true;
        auto wait_for = [&](uint64_t* bar, int parity) { return (bool)__all_sync(0xffffffffu, kvp_wait(bar, parity & 1, &s_fail)); };
#pragma unroll 1
        for (int j = 0; j < mine; j++) {
            ok = wait_for(&s_full[tile][j & 1], j >> 1);
            if (!ok) break;
            tc_fence_after();
            const uint32_t ts = tmem + lanes + 128 * tile + 64 * (j & 1);   // S, then P
            const KvpMeta& me = s_meta[j & 7];   // written before the tile's K was announced
            const int key0 = j * kKvpTile;
            uint32_t x[2][32];
            tmem_ld64(ts, x);
            // some row of the warp does not see every key of the tile
            if (__any_sync(0xffffffffu, key0 + kKvpTile - 1 > lim) || me.live != 0xFu) {
#pragma unroll
                for (int b = 0; b < 2; b++) {   // -inf at the keys that are not seen
                    const int n = lim - (key0 + 32 * b) + 1;
                    uint32_t see = n >= 32 ? 0xFFFFFFFFu : n <= 0 ? 0u : (1u << n) - 1u;
                    if (!((me.live >> (2 * b)) & 1)) see &= 0xFFFF0000u;
                    if (!((me.live >> (2 * b + 1)) & 1)) see &= 0xFFFFu;
#pragma unroll
                    for (int e = 0; e < 32; e++) x[b][e] = (see >> e) & 1 ? x[b][e] : 0xFF800000u;
                }
            }
            // factors of the scores: never 0, so that -inf stays -inf
            float cs[4];
#pragma unroll
            for (int g = 0; g < 4; g++) cs[g] = fmaxf(me.ks[g] * rs, 1.17549435e-38f);
            // ---- the tile's maximum
            float mt = -INFINITY;
#pragma unroll
            for (int g = 0; g < 4; g++) {
                const uint32_t* v = x[g >> 1] + 16 * (g & 1);
                float mx = __uint_as_float(v[0]);
#pragma unroll
                for (int e = 1; e < 15; e += 2) mx = max3(mx, __uint_as_float(v[e]), __uint_as_float(v[e + 1]));
                mx = fmaxf(mx, __uint_as_float(v[15]));
                mt = fmaxf(mt, fmaf(mx, cs[g], me.lv[g]));   // fmaxf leaves a NaN out: m is never one
            }
            // the reference follows the maximum in steps of more than 8
            const bool grow = mt > m + 8.0f;
            if (__any_sync(0xffffffffu, grow)) {
                const float f = grow ? (m == -INFINITY ? 0.0f : kv_exp2(m - mt)) : 1.0f;
                if (grow) m = mt;
                l *= f;
                if (j > 0) {
                    ok = wait_for(&pv_done[tile], j - 1);   // O is whole up to the tile before
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll 1
                    for (int b = 0; b < c.hd; b += 16) {
                        float o[16];
                        uint32_t u[16];
                        tmem_ld16(to + b, o);
#pragma unroll
                        for (int e = 0; e < 16; e++) u[e] = __float_as_uint(o[e] * f);
                        tmem_st16(to + b, u);
                    }
                }
            }
            // ---- weights
            const float ref = m == -INFINITY ? 0.0f : m;
            const uint64_t ref2 = f2_pack(-ref, -ref);
            uint64_t sum[2] = {0, 0};
#pragma unroll
            for (int b = 0; b < 2; b++) {
                uint32_t p[16], pl[16];
#pragma unroll
                for (int g = 0; g < 2; g++) {
                    const float fv = me.fv[2 * b + g];
                    const uint64_t cs2 = f2_pack(cs[2 * b + g], cs[2 * b + g]), fv2 = f2_pack(fv, fv);
#pragma unroll
                    for (int e = 0; e < 16; e += 2) {
                        float2 w = f2_unpack(f2_fma(
                            f2_pack(__uint_as_float(x[b][16 * g + e]), __uint_as_float(x[b][16 * g + e + 1])), cs2, ref2));
                        const uint64_t w2 = f2_pack(kv_exp2(w.x), kv_exp2(w.y));
                        sum[g] = f2_add(sum[g], w2);
                        w = f2_unpack(f2_mul(w2, fv2));
                        p[8 * g + e / 2] = half2_bits(w.x, w.y);
                        if (TERMS == 2) {
                            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&p[8 * g + e / 2]));
                            pl[8 * g + e / 2] = half2_bits(w.x - f.x, w.y - f.y);
                        }
                    }
                }
                tmem_st16(ts + 16 * b, p);
                if (TERMS == 2) tmem_st16(ts + 32 + 16 * b, pl);
            }
            const float2 s0 = f2_unpack(sum[0]), s1 = f2_unpack(sum[1]);
            l += (s0.x + s0.y) + (s1.x + s1.y);
            if (me.nan) {   // a NaN scale reaches the rows that see a key under it
#pragma unroll 1
                for (int g = 0; g < 4; g++)
                    if (((me.nan >> g) & 1) && key0 + 16 * g <= lim) l = __int_as_float(0x7FC00000);
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_addr(&p_full[tile][j & 1]));
        }
        if (bad && l != 0.0f) l = __int_as_float(0x7FC00000);   // a query that is not finite, unless it sees nothing
        // ---- out = O / (2^7 l) vref, in this order: vref may be near the end of the range
        if (ok && mine > 0) ok = wait_for(&o_full[tile], 0);
        tc_fence_after();
        if (ok && (tile < nq)) {
            const float f = l == 0.0f ? 0.0f : 0.0078125f / l;
            T* dst = (T*)a.out + (q.t0 + tok) * a.out_stride + (long long)head * c.hd;
            if (a.vec_out) {
                // Through the place of the tile's queries, which no MMA reads any more, 16 bytes a piece: a store then
                // covers whole rows (a thread's own row is 16-byte pieces of 32 rows to a store).
                constexpr int PR = 128 * (int)sizeof(T) / 16, RI = 32 / PR;   // pieces of a row, rows a store
                constexpr int PV = 16 / (int)sizeof(T);                       // values of a piece
                unsigned char* st = qs + tile * TERMS * kKvpQ + (warp & 3) * 32 * PR * 16;
                // without keys no MMA has waited for all four warps' queries
                if (mine == 0) asm volatile("bar.sync %0, 128;" ::"r"(1 + tile) : "memory");
#pragma unroll 1
                for (int b = 0; b < c.hd; b += 16) {
                    float x[16];
                    if (mine > 0) tmem_ld16(to + b, x);
#pragma unroll
                    for (int e = 0; e < 16; e++) x[e] = l == 0.0f || mine == 0 ? 0.0f : x[e] * f * vref;
#pragma unroll
                    for (int e = 0; e < 16 / PV; e++) {
                        T y[PV];
#pragma unroll
                        for (int i = 0; i < PV; i++) y[i] = from_f32<T>(x[PV * e + i]);
                        *reinterpret_cast<uint4*>(st + lane * PR * 16 + (((b / PV + e) ^ (lane & (PR - 1))) << 4)) =
                            *reinterpret_cast<const uint4*>(y);
                    }
                }
                __syncwarp();
                const long long at = live_row ? dst - (T*)a.out : -1;
                const int piece = lane & (PR - 1);
                const bool in = piece * PV < c.hd;
#pragma unroll 4
                for (int r0 = 0; r0 < 32; r0 += RI) {
                    const int row = r0 + lane / PR;
                    const long long to_row = __shfl_sync(0xffffffffu, at, row);
                    const uint4 y = *reinterpret_cast<const uint4*>(st + row * PR * 16 + ((piece ^ (row & (PR - 1))) << 4));
                    if (to_row >= 0 && in) *reinterpret_cast<uint4*>((T*)a.out + to_row + piece * PV) = y;
                }
            } else {
#pragma unroll 1
                for (int b = 0; b < c.hd; b += 16) {
                    float x[16];
                    if (mine > 0) tmem_ld16(to + b, x);
#pragma unroll
                    for (int e = 0; e < 16; e++) x[e] = l == 0.0f || mine == 0 ? 0.0f : x[e] * f * vref;
                    if (live_row) store16(dst + b, false, x);
                }
            }
        }
        tc_fence_before();
    } else if (warp < 16) {
        // ================= K or V to fp16 =================
        regs_less<kKvpRegsConv>();
        const bool is_k = (warp & 2) == 0;
        const int w4 = (warp & 1) | ((warp >> 1) & 2), id = 32 * w4 + lane;   // of the four warps of K, or of V
        // Lane e (mod 4) keeps track of keys 64 j + 16 e..+15 of a tile.  Values are fetched two tiles ahead, pages three.
        auto look = [&](int j) {
            const int pos = j * kKvpTile + 16 * (lane & 3);
            return j < ntiles && pos < q.len ? table[pos >> c.page_log] : -1;
        };
        // (page, head) of the lane's 16 keys, or -1
        auto unit_of = [&](int j, int page) {
            const int pos = j * kKvpTile + 16 * (lane & 3);
            if (j >= ntiles || pos >= q.len) return -1LL;
            if (page < 0 || page >= c.n_pages) {
                kv_flag(c, KV_BAD_PAGE);
                return -1LL;
            }
            return (long long)page * c.nkv + h;
        };
        // where the values of its 16 keys lie, or -1
        auto at_of = [&](int j, long long unit) {
            return unit < 0 ? -1LL : (unit * c.page + ((j * kKvpTile + 16 * (lane & 3)) & (c.page - 1))) * c.hd;
        };
        if (is_k) {
            const int kr = id >> 3, kc = id & 7;   // row of each 16, 16 dimensions
            const bool in = 16 * kc < c.hd;
            const int8_t* src = c.k + a.layer * c.plane() + kr * c.hd + 16 * kc;
            const float* scales = ((lane & 4) ? c.v_scale : c.k_scale) + (long long)a.layer * c.n_pages * c.nkv;
            // 1 / vref in two factors, since a small vref's is past fp32's range: 1 or 2^64, and what is left
            const float vinv0 = vref < 1.0f ? 18446744073709551616.0f : 1.0f, vinv1 = vref > 0.0f ? 1.0f / (vref * vinv0) : 0.0f;
            unsigned char *mine = raw + 16 * id;   // the thread's pieces, 2 KB apart
            unsigned char *to0 = kst + kvp_piece(64, kr, 2 * kc), *to1 = kst + kvp_piece(64, kr, 2 * kc + 1);   // + 2 KB every 16 rows
            auto fetch = [&](int j, int page) {
                const long long unit = unit_of(j, page), at0 = at_of(j, unit);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const long long at = __shfl_sync(0xffffffffu, at0, e);
                    if (at >= 0 && in) cp_async16(mine + (j & 1) * kKvpRaw + 2048 * e, src + at);
                }
                if (w4 == 0 && lane < 8) {
                    float* to = &s_scale[j & 1][lane];
                    if (unit >= 0)
                        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_addr(to)), "l"(scales + unit) : "memory");
                    else
                        *to = -1.0f;
                }
                cp_async_commit();
            };
            fetch(0, look(0));
            fetch(1, look(1));
            int page = look(2);
#pragma unroll 1
            for (int j = 0; j < ntiles; j++) {
                const int st = j % ST;
                cp_async_wait<1>();
                if (j >= ST && !kvp_wait(&k_empty[st], (j / ST - 1) & 1, &s_fail)) break;
                if (in) {
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const uint4 x = *reinterpret_cast<const uint4*>(mine + (j & 1) * kKvpRaw + 2048 * e);
                        const uint2 p0 = int8x4_to_half(x.x), p1 = int8x4_to_half(x.y), p2 = int8x4_to_half(x.z),
                                    p3 = int8x4_to_half(x.w);
                        *reinterpret_cast<uint4*>(to0 + st * kKvpStage + e * 2048) = make_uint4(p0.x, p0.y, p1.x, p1.y);
                        *reinterpret_cast<uint4*>(to1 + st * kKvpStage + e * 2048) = make_uint4(p2.x, p2.y, p3.x, p3.y);
                    }
                }
                // Words of tile j - 8: k_empty says that S of tile j - ST (4 at most) was issued, which P of the tile
                // two before that preceded, so the softmax of both row tiles is past it.
                if (w4 == 0) {
                    __syncwarp();   // the scales that lanes 0..7 copied
                    const float ks = s_scale[j & 1][lane & 3], vs = s_scale[j & 1][4 + (lane & 3)];
                    KvpMeta& me = s_meta[j & 7];
                    const unsigned live = __ballot_sync(0xffffffffu, ks != -1.0f);
                    const unsigned nan = __ballot_sync(0xffffffffu, ks != ks || vs != vs);
                    if (lane < 4) {
                        me.ks[lane] = ks >= 0.0f ? ks : 1.0f;
                        const float part = vs > 0.0f ? vs * vinv0 * vinv1 : 0.0f;
                        me.fv[lane] = 128.0f * part;
                        me.lv[lane] = fmaxf(__log2f(part), kKvpLvMin);
                    }
                    if (lane == 0) {
                        me.live = live & 0xF;
                        me.nan = nan & 0xF;
                    }
                }
                fence_smem_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_addr(&k_full[st]));
                fetch(j + 2, page);
                page = look(j + 3);
            }
        } else {
            const int tg = lane & 7, vd = 8 * ((lane >> 3) + 4 * w4);   // 8 tokens, 8 dimensions
            const bool in = vd < c.hd;
            const int8_t* src = c.v + a.layer * c.plane() + (8 * tg & 15) * c.hd + vd;
            unsigned char *mine = raw + 2 * kKvpRaw + 8 * id;   // the thread's pieces, 1 KB apart
            unsigned char* to = vst + vd * 128;
            auto fetch = [&](int j, int page) {
                const long long at = __shfl_sync(0xffffffffu, at_of(j, unit_of(j, page)), tg >> 1);
                if (at >= 0 && in) {
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(
                                         smem_addr(mine + (j & 1) * kKvpRaw + 1024 * e)),
                                     "l"(src + at + e * c.hd)
                                     : "memory");
                }
                cp_async_commit();
            };
            fetch(0, look(0));
            fetch(1, look(1));
            int page = look(2);
#pragma unroll 1
            for (int j = 0; j < ntiles; j++) {
                const int st = j % ST;
                cp_async_wait<1>();
                if (j >= ST && !kvp_wait(&v_empty[st], (j / ST - 1) & 1, &s_fail)) break;
                if (in) {
                    uint2 x[8];
#pragma unroll
                    for (int e = 0; e < 8; e++) x[e] = *reinterpret_cast<const uint2*>(mine + (j & 1) * kKvpRaw + 1024 * e);
#pragma unroll
                    for (int w = 0; w < 2; w++) {
                        uint32_t lo[4], hi[4];   // dimension vd + 4 w + d: tokens 0..3, 4..7 of the eight
                        auto word = [&](int e) { return w ? x[e].y : x[e].x; };
                        transpose4(word(0), word(1), word(2), word(3), lo);
                        transpose4(word(4), word(5), word(6), word(7), hi);
#pragma unroll
                        for (int d = 0; d < 4; d++) {   // vd is a multiple of 8: row & 7 is 4 w + d
                            const uint2 p0 = int8x4_to_half(lo[d]), p1 = int8x4_to_half(hi[d]);
                            *reinterpret_cast<uint4*>(to + st * kKvpStage + (4 * w + d) * 128 + ((tg ^ (4 * w + d)) << 4)) =
                                make_uint4(p0.x, p0.y, p1.x, p1.y);
                        }
                    }
                }
                fence_smem_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_addr(&v_full[st]));
                fetch(j + 2, page);
                page = look(j + 3);
            }
        }
        cp_async_wait<0>();
    } else {
        // ================= MMA issue, row tile t =================
        regs_less<kKvpRegsMma>();
        const int t = warp - 16, mine = t < NQ ? nt[t & 1] : 0;
        if (t < NQ) {
            // Descriptors count in 16 bytes; a k-step of 16 values is 2.
            const uint32_t id_s = kvp_idesc(kKvpTile), id_o = kvp_idesc(c.hd);
            const uint32_t qd = umma_lo(smem_addr(qs)), kd = umma_lo(smem_addr(kst)), vd = umma_lo(smem_addr(vst));
            const int nk = c.hd / 16;
            auto scores = [&](int j) {
                const uint32_t d = tmem + 128 * t + 64 * (j & 1), kb = kd + (j % ST) * (kKvpStage >> 4);
#pragma unroll
                for (int term = 0; term < TERMS; term++)
                    umma_run_ss(d, qd + (t * TERMS + term) * (kKvpQ >> 4), kb, kKvpQ >> 5, kKvpStage >> 5, id_s, nk, term);
                umma_commit_warp(smem_addr(&s_full[t][j & 1]));
            };
            auto values = [&](int j) {
                const uint32_t d = tmem + 256 + 128 * t, p = tmem + 128 * t + 64 * (j & 1), vb = vd + (j % ST) * (kKvpStage >> 4);
#pragma unroll
                for (int term = 0; term < TERMS; term++) umma_run4_ts(d, p + 32 * term, vb, id_o, term != 0 || j > 0);
                umma_commit_warp(smem_addr(&pv_done[t]));
            };
            auto wait_for = [&](uint64_t* bar, int parity) { return kvp_wait(bar, parity & 1, &s_fail); };
            // A wait that gives up is looked at once a turn: what is issued until then has no reader.
            bool ok = ntiles == 0 || wait_for(&q_full, 0);
            for (int j = 0; j < 2 && j < ntiles; j++) {
                ok = wait_for(&k_full[j], 0) && ok;
                tc_fence_after();
                __syncwarp();
                if (j < mine) scores(j);
                umma_commit_warp(smem_addr(&k_empty[j]));
            }
#pragma unroll 1
            for (int j = 0; j < ntiles && __all_sync(0xffffffffu, ok); j++) {
                // a warp past its own tiles goes on at the others' pace, so that its commits count for the right tile
                ok = wait_for(&v_full[j % ST], j / ST) && ok;
                if (j < mine) ok = wait_for(&p_full[t][j & 1], j >> 1) && ok;
                tc_fence_after();
                __syncwarp();
                if (j < mine) values(j);
                if (j == mine - 1) umma_commit_warp(smem_addr(&o_full[t]));
                umma_commit_warp(smem_addr(&v_empty[j % ST]));
                if (j + 2 >= ntiles) continue;
                ok = wait_for(&k_full[(j + 2) % ST], (j + 2) / ST) && ok;
                if (j + 2 < mine) ok = wait_for(&pv_done[t], j) && ok;   // P of tile j lies where this S goes
                tc_fence_after();
                __syncwarp();
                if (j + 2 < mine) scores(j + 2);
                umma_commit_warp(smem_addr(&k_empty[(j + 2) % ST]));
            }
            umma_commit_warp(smem_addr(&done_bar));
        } else if (blockIdx.x == 0) {
            kv_vet_rows(c, a.r, threadIdx.x - 32 * (16 + NQ), 32 * (4 - NQ));
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 16) {
        mbar_wait(smem_addr(&done_bar), 0, 1u << 20);   // every MMA issued is complete
        __syncwarp();
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
    if (threadIdx.x == 0 && s_fail) kv_flag(c, KV_TIMEOUT);
}

}  // namespace aion
