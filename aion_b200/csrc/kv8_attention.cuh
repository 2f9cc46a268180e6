// Attention over the 8-bit paged K/V cache (kv8.cuh).
#pragma once

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
};

// One warp a (row, head): an online softmax over the positions in fp32.
constexpr int kKvAttnThreads = 128;
template <typename T>
__global__ void __launch_bounds__(kKvAttnThreads) k_kv_attention(KvAttnArgs a) {
    const KvView& c = a.c;
    const int lane = threadIdx.x & 31, row = blockIdx.x, h = blockIdx.y * (kKvAttnThreads / 32) + (threadIdx.x >> 5);
    if (h >= a.n_heads) return;
    int s = row;
    if (a.r.cu) {
        int lo = 0, hi = a.r.n_seq - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (a.r.cu[mid] <= row) lo = mid;
            else hi = mid - 1;
        }
        s = lo;
        if (row < a.r.cu[s] || row >= a.r.cu[s + 1]) return;
    }
    const int p0 = a.r.pos0[s], slot = a.r.seqs[s], kvh = h / a.group;
    const T* q = (const T*)a.q + row * a.q_stride + (long long)h * c.hd;
    float x[4], o[4] = {0, 0, 0, 0}, m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; e++) x[e] = lane + 32 * e < c.hd ? to_f32(q[lane + 32 * e]) * a.scale : 0.0f;
    const bool held = slot >= 0 && slot < c.max_seqs;
    if (!held && p0 >= 0 && lane == 0) kv_flag(c, KV_BAD_ARG);
    const long long end = !held || p0 < 0 ? 0 : (long long)p0 + (row - a.r.begin(s)) + 1;
    for (long long j = 0; j < end; j++) {
        const long long pg = j >> c.page_log;
        const int page = pg < c.max_pages ? c.tables[(size_t)slot * c.max_pages + pg] : -1;
        if (page < 0 || page >= c.n_pages) {
            if (lane == 0) kv_flag(c, KV_BAD_PAGE);
            if (pg >= c.max_pages) break;
            continue;
        }
        const long long at = a.layer * c.plane() + (((long long)page * c.nkv + kvh) * c.page + (j & (c.page - 1))) * c.hd;
        const long long sc = ((long long)a.layer * c.n_pages + page) * c.nkv + kvh;
        float d = 0.0f;
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (lane + 32 * e < c.hd) d += x[e] * (float)c.k[at + lane + 32 * e];
        d = warp_sum(d) * c.k_scale[sc];
        const float mn = fmaxf(m, d), al = m == -INFINITY ? 0.0f : exp2f(m - mn);
        const float p = exp2f(d - mn), pv = p * c.v_scale[sc];
        l = l * al + p;
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (lane + 32 * e < c.hd) o[e] = o[e] * al + pv * (float)c.v[at + lane + 32 * e];
        m = mn;
    }
    T* out = (T*)a.out + row * a.out_stride + (long long)h * c.hd;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int e = 0; e < 4; e++)
        if (lane + 32 * e < c.hd) out[lane + 32 * e] = from_f32<T>(o[e] * inv);
}

}  // namespace aion
