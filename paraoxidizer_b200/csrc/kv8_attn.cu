// kv8_attn.cu -- attention over int8 pages with one scale per page, kv head and side.
#include "kv8_attn.h"

namespace pox {

// One CTA of 128 threads per (row, query head): tiles of 128 tokens, one token's score per thread, then
// one dim's sum per thread, with the running maximum and sum of the softmax.
template <int HD, typename T>
__global__ void __launch_bounds__(128) kv8_attn_rows_kernel(Kv8Attn<T> a) {
    const uint32_t nh = (uint32_t)(a.G * a.c.kvh), r = blockIdx.x / nh, qh = blockIdx.x % nh, h = qh / a.G;
    const int tid = threadIdx.x;
    __shared__ float qs[HD], ps[128], red[4];
    __shared__ float svs[8];
    __shared__ int blks[8];
    const uint32_t s = a.b.row_starts ? find_seq(a.b, r, 0, 1) : r;
    SeqSpan sp;
    if (!seq_span(a.b, s, sp, a.err)) return;
    const int pos = sp.ctx - sp.n + (int)(r - sp.r0);
    for (int d = tid; d < HD; d += 128) qs[d] = to_f32(a.q.at(r, qh)[d]) * a.scale;
    float m = -INFINITY, l = 0.f, acc = 0.f;
    for (int t0 = 0; t0 <= pos; t0 += 128) {
        __syncthreads();
        if (tid < 8) {
            const int page = t0 / kPage + tid;
            int blk = page * kPage <= pos ? a.b.btab[(size_t)s * a.b.mbps + page] : -1;
            if (page * kPage <= pos && (blk < 0 || (uint32_t)blk >= a.c.num_blocks)) {
                atomicOr(a.err, kErrAttnPage);
                blk = -1;
            }
            blks[tid] = blk;
            svs[tid] = blk >= 0 ? a.c.scales[((size_t)blk * a.c.kvh + h) * 2 + 1] : 0.f;
        }
        __syncthreads();
        const int t = t0 + tid, blk = blks[tid / kPage];
        float sc = -INFINITY;
        if (t <= pos && blk >= 0) {
            const size_t pg = (size_t)blk * a.c.kvh + h;
            const int8_t* k = a.c.pages + pg * (2 * kPage * HD);
            float dot = 0.f;
            for (int d = 0; d < HD; d++) dot = fmaf(qs[d], (float)k[kv8_k_off<HD>(t % kPage, d)], dot);
            sc = dot * a.c.scales[pg * 2];
        }
        const float wm = warp_max(sc);
        if ((tid & 31) == 0) red[tid >> 5] = wm;
        __syncthreads();
        const float mt = fmaxf(m, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
        const float ref = mt == -INFINITY ? 0.f : mt, p = expf(sc - ref);
        ps[tid] = p;
        const float ws = warp_sum(p);
        __syncthreads();
        if ((tid & 31) == 0) red[tid >> 5] = ws;
        __syncthreads();
        const float f = m == -INFINITY ? 0.f : expf(m - ref);
        l = l * f + ((red[0] + red[1]) + (red[2] + red[3]));
        m = mt;
        acc *= f;
        if (tid < HD)
            for (int j = 0; j < 128 && t0 + j <= pos; j++) {
                const int b = blks[j / kPage];
                if (b < 0) continue;
                const int8_t* pg = a.c.pages + ((size_t)b * a.c.kvh + h) * (2 * kPage * HD);
                acc = fmaf(ps[j] * svs[j / kPage], (float)pg[kv8_v_off<HD>(j % kPage, tid)], acc);
            }
    }
    if (tid < HD) a.out.at(r, qh)[tid] = from_f32<T>(l > 0.f ? acc / l : l == 0.f ? 0.f : l);
}

template <int HD, typename T>
cudaError_t launch_kv8_attention(const Kv8Attn<T>& a, cudaStream_t st) {
    kv8_attn_rows_kernel<HD, T><<<a.b.rows * (unsigned)(a.G * a.c.kvh), 128, 0, st>>>(a);
    return cudaGetLastError();
}

#define POX_KV8_ATTN(HD)                                                                     \
    template cudaError_t launch_kv8_attention<HD, float>(const Kv8Attn<float>&, cudaStream_t);   \
    template cudaError_t launch_kv8_attention<HD, __half>(const Kv8Attn<__half>&, cudaStream_t); \
    template cudaError_t launch_kv8_attention<HD, __nv_bfloat16>(const Kv8Attn<__nv_bfloat16>&, cudaStream_t);
POX_KV8_ATTN(32)
POX_KV8_ATTN(64)
POX_KV8_ATTN(128)

}  // namespace pox
