// kv8_attn.cu -- attention of few rows over int8 pages with one scale per page, kv head and side.
//
// For row r (a query head at a token) of one kv head, with page scales a (of k) and b (of v):
//   s_t = scale log2(e) a q . k_t,   u_t = s_t + log2 b,   p_t = 2^(u_t - m),   m about max u_t
//   out = sum_t p_t v_t / sum_t p_t / b
// where k_t and v_t are the stored whole numbers. Taking the maximum over u instead of s puts the scale of
// v into the exponent: the products see whole numbers and p <= 2^8, and no page's scale multiplies a tile.
#include "kv8_attn.h"
#include "kv8_math.cuh"

namespace pox {

constexpr int kStepStages = 4;  // pages in flight per warp

// One CTA per (sequence, kv head, split of the context, tile of rows). Each warp streams whole pages (K and V of 16
// tokens of the kv head, 32 HD contiguous bytes) through a ring of its own with one bulk copy a page, and runs both products on
// mma.sync m16n8k16 with f32 accumulators: the rows are A, the int8 operands become exact f16 on the way from
// shared memory. An MMA does not care in which order k runs, so the order is the one that the page's bytes
// have: lane (g, t) takes 16 dims of a token for Q K^T and the four tokens 4 t .. 4 t + 3 of a dim for P V, and
// the scores leave the first product where the second wants them.
// PAIR: 8 rows, A rows g and g + 8 being the two f16 terms of row g (f32 rows need them; fewer rows
// than 9 leave the place free). Otherwise 16 rows, p rounded to f16 (2^-11 of p, as the output's type).
template <int HD, typename T, bool PAIR>
__global__ void __launch_bounds__(32 * kStepWarps, 3) kv8_attn_step_kernel(Kv8Attn<T> a, Kv8StepPlan p) {
    constexpr int RT = PAIR ? 8 : 16, KW = HD / 16, NJ = HD / 8, PB = 32 * HD, NR = PAIR ? 1 : 2;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ __align__(8) uint64_t bars[kStepWarps][kStepStages];
    __shared__ float ml[kStepWarps][2][RT];
    __shared__ uint32_t last_cta;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    uint32_t bi = blockIdx.x;
    const int rt = bi % p.row_tiles;
    bi /= p.row_tiles;
    const int sp = bi % p.splits;
    bi /= p.splits;
    const int h = bi % a.c.kvh;
    const uint32_t s = bi / a.c.kvh;
    SeqSpan sq;
    if (!seq_span(a.b, s, sq, a.err)) return;
    const int rows = sq.n * a.G, row0 = rt * RT;
    if (row0 >= rows || rows > p.most_rows) return;
    const int pos0 = sq.ctx - sq.n, pmin = pos0 + row0 / a.G, pmax = pos0 + (min(row0 + RT, rows) - 1) / a.G;
    const int pages = pmax < 0 ? 0 : pmax / kPage + 1;
    const int ns = max(1, (pages + p.pages_per_split - 1) / p.pages_per_split);
    if (sp >= ns) return;

    // this warp's pages: first, first + W, ..; lane i holds the i-th one's place and scales
    const int first = sp * p.pages_per_split + warp, end = min(pages, (sp + 1) * p.pages_per_split);
    const int cnt = first < end ? (end - first + kStepWarps - 1) / kStepWarps : 0;
    const uint32_t ring = smem_u32(smem) + warp * kStepStages * PB, bar = smem_u32(&bars[warp][0]);
    if (lane == 0) {
        for (int i = 0; i < kStepStages; i++) mbar_init(bar + 8 * i, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    size_t place = 0;
    bool there = false;
    if (lane < cnt) {
        const int blk = a.b.btab[(size_t)s * a.b.mbps + first + lane * kStepWarps];
        there = blk >= 0 && (uint32_t)blk < a.c.num_blocks;
        if (!there) atomicOr(a.err, kErrAttnPage);
        place = there ? (size_t)blk * a.c.kvh + h : 0;
    }
    const unsigned there_m = __ballot_sync(0xffffffffu, there);
    auto fetch = [&](int i) {  // page i of this warp into its stage (a page out of range: page 0, unread)
        const size_t pl = __shfl_sync(0xffffffffu, (unsigned long long)place, i);
        if (lane == 0) {
            const int st = i % kStepStages;
            mbar_expect_tx(bar + 8 * st, PB);
            bulk_g2s(ring + st * PB, a.c.pages + pl * PB, PB, bar + 8 * st);
        }
    };
    for (int i = 0; i < min(cnt, kStepStages); i++) fetch(i);
    const float2 ab = lane < cnt ? *reinterpret_cast<const float2*>(a.c.scales + place * 2) : make_float2(0.f, 0.f);
    // log2 b; a scale of 0 stands for zeros whatever the bytes: 1e-30 of them is nothing next to any other page
    const float lb = log2f(fmaxf(ab.y, 1e-30f) + (ab.y - ab.y)), ib = 1.0f / fmaxf(ab.y, 1e-30f);

    // A fragments of the rows, and what takes their products to scores
    uint32_t qa[KW][4];
    float qf[NR];
    int rpos[NR];
#pragma unroll
    for (int r = 0; r < NR; r++) {
        const int row = row0 + g + 8 * r;
        const bool ok = row < rows;
        rpos[r] = ok ? pos0 + row / a.G : 0;
        const T* q = a.q.at((size_t)sq.r0 + (ok ? row / a.G : 0), h * a.G + (ok ? row % a.G : 0));
        float v[KW][4], m = 0.f;
#pragma unroll
        for (int w = 0; w < KW; w++) {
            const int d = HD == 32 ? 8 * t + 4 * w : 64 * (w / 4) + 16 * t + 4 * (w % 4);
            if (ok) load4(q + d, a.vec, v[w]);
            else v[w][0] = v[w][1] = v[w][2] = v[w][3] = 0.f;
#pragma unroll
            for (int i = 0; i < 4; i++) m = fmaxf(m, fabsf(v[w][i]));
        }
        float f = 1.f, inv = 1.f;
        if constexpr (sizeof(T) == 4 || std::is_same<T, __nv_bfloat16>::value) {
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
            f = row_factor(m, inv);
        }
        qf[r] = inv * a.scale;
#pragma unroll
        for (int w = 0; w < KW; w++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const float x = v[w][2 * i] * f, y = v[w][2 * i + 1] * f;
                qa[w][2 * i + r] = pack_f16(x, y);
                if constexpr (PAIR && sizeof(T) == 4) {
                    const float2 hi = unpack_f16(qa[w][2 * i]);
                    qa[w][2 * i + 1] = pack_f16(x - hi.x, y - hi.y);
                } else if (PAIR) {
                    qa[w][2 * i + 1] = 0u;
                }
            }
    }

    float o[NJ][4], m[NR], l[NR];
#pragma unroll
    for (int j = 0; j < NJ; j++) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
#pragma unroll
    for (int r = 0; r < NR; r++) m[r] = -INFINITY, l[r] = 0.f;
    bool bad = false;
    for (int i = 0; i < cnt; i++) {
        const int st = i % kStepStages, page = first + i * kStepWarps;
        const uint32_t base = ring + st * PB;
        if (!bad) bad = __any_sync(0xffffffffu, !mbar_wait(bar + 8 * st, (i / kStepStages) & 1));
        const float pa = __shfl_sync(0xffffffffu, ab.x, i), pl = __shfl_sync(0xffffffffu, lb, i),
                    pi = __shfl_sync(0xffffffffu, ib, i);
        float sc[2][4];
#pragma unroll
        for (int nb = 0; nb < 2; nb++) {
            const int tok = 4 * (g >> 1) + 2 * nb + (g & 1);
            sc[nb][0] = sc[nb][1] = sc[nb][2] = sc[nb][3] = 0.f;
            uint32_t kw[KW];
            if constexpr (HD == 32) {
                const uint2 x = lds64(base + tok * HD + 8 * t);
                kw[0] = x.x, kw[1] = x.y;
            } else {
#pragma unroll
                for (int c = 0; c < HD / 64; c++) {
                    const uint4 x = lds128(base + tok * HD + (HD == 128 ? (64 * c + 16 * t) ^ ((g & 1) << 6) : 16 * t));
                    kw[4 * c] = x.x, kw[4 * c + 1] = x.y, kw[4 * c + 2] = x.z, kw[4 * c + 3] = x.w;
                }
            }
#pragma unroll
            for (int w = 0; w < KW; w++) {
                uint32_t b0, b1;
                i8x4_to_f16x4(kw[w], b0, b1);
                mma_16816(sc[nb], qa[w][0], qa[w][1], qa[w][2], qa[w][3], b0, b1);
            }
        }
        // u of tokens 4 t + 2 nb + e
        const bool whole = page * kPage + kPage - 1 <= pmin && (there_m >> i & 1);
        float u[NR][4], mx[NR];
        bool grow = false;
#pragma unroll
        for (int r = 0; r < NR; r++) {
            const float f = qf[r] * pa;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float x = PAIR ? sc[e >> 1][e & 1] + sc[e >> 1][2 + (e & 1)] : sc[e >> 1][2 * r + (e & 1)];
                u[r][e] = fmaf(x, f, pl);
                if (!whole && (page * kPage + 4 * t + e > rpos[r] || !(there_m >> i & 1))) u[r][e] = -INFINITY;
            }
            float y = fmaxf(fmaxf(u[r][0], u[r][1]), fmaxf(u[r][2], u[r][3]));
            y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 1));
            mx[r] = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 2));
            grow |= mx[r] > m[r] + 8.0f;
        }
        // the reference moves only when p would pass 2^8: after the first pages it hardly ever does
        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
            for (int r = 0; r < NR; r++) {
                const float to = mx[r] > m[r] + 8.0f ? mx[r] : m[r];
                const float f = m[r] == -INFINITY ? (to == -INFINITY ? 1.f : 0.f) : ex2(m[r] - to);
                m[r] = to;
                l[r] *= f;
#pragma unroll
                for (int j = 0; j < NJ; j++) {
                    o[j][2 * r] *= f, o[j][2 * r + 1] *= f;
                    if (PAIR) o[j][2] *= f, o[j][3] *= f;
                }
            }
        }
        uint32_t pp[4];  // A fragment of P: tokens 4 t, 4 t + 1 | 4 t + 2, 4 t + 3
#pragma unroll
        for (int r = 0; r < NR; r++) {
            const float ref = m[r] == -INFINITY ? 0.f : m[r];
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; e++) x[e] = ex2(u[r][e] - ref);
            const float sum = (x[0] + x[1]) + (x[2] + x[3]);
            if (sum != 0.f) l[r] = fmaf(sum, pi, l[r]);  // (an unseen page's scale may be anything)
            pp[r] = pack_f16(x[0], x[1]);
            pp[2 + r] = pack_f16(x[2], x[3]);
            if (PAIR) {
                const float2 h0 = unpack_f16(pp[0]), h1 = unpack_f16(pp[2]);
                pp[1] = pack_f16(x[0] - h0.x, x[1] - h0.y);
                pp[3] = pack_f16(x[2] - h1.x, x[3] - h1.y);
            }
        }
#pragma unroll
        for (int j = 0; j < NJ; j++) {
            uint32_t w, b0, b1;
            asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w) : "r"(base + kPage * HD + (8 * j + g) * kPage + 4 * t));
            i8x4_to_f16x4(w, b0, b1);
            mma_16816(o[j], pp[0], pp[1], pp[2], pp[3], b0, b1);
        }
        __syncwarp();  // every lane has read the stage
        if (i + kStepStages < cnt && !bad) fetch(i + kStepStages);
        if (bad) {  // a copy did not come in time: give the ones in flight as long again, and leave
            for (int k = i; k < min(cnt, i + kStepStages); k++) mbar_wait(bar + 8 * (k % kStepStages), (k / kStepStages) & 1);
            if (lane == 0) atomicOr(a.err, kErrWaitRing);
            break;
        }
    }

    // the warps' parts: (m, l) and o in units of 2^m, through the ring's space
#pragma unroll
    for (int r = 0; r < NR; r++) {
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
        if (t == 0) ml[warp][0][g + 8 * r] = m[r], ml[warp][1][g + 8 * r] = l[r];
    }
    __syncthreads();
    float* os = reinterpret_cast<float*>(smem);  // [warp][RT][HD]
#pragma unroll
    for (int j = 0; j < NJ; j++)
#pragma unroll
        for (int r = 0; r < NR; r++) {
            const float2 x = PAIR ? make_float2(o[j][0] + o[j][2], o[j][1] + o[j][3])
                                  : make_float2(o[j][2 * r], o[j][2 * r + 1]);
            *reinterpret_cast<float2*>(os + ((size_t)warp * RT + g + 8 * r) * HD + 8 * j + 2 * t) = x;
        }
    __syncthreads();
    const size_t item = ((size_t)s * a.c.kvh + h) * p.row_tiles + rt;
    float* part = p.part + (item * p.splits + sp) * RT * (HD + 2);
    const int valid = min(RT, rows - row0);
    for (int i = tid; i < valid * (HD / 4); i += 32 * kStepWarps) {
        const int r = i / (HD / 4), d = 4 * (i % (HD / 4));
        float M = -INFINITY, L = 0.f;
#pragma unroll
        for (int w = 0; w < kStepWarps; w++) M = fmaxf(M, ml[w][0][r]);
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kStepWarps; w++) {
            // NaN scores leave m at -inf with l NaN: the weight of such a part is 1, so that the row is NaN
            const float f = ml[w][0][r] == -INFINITY ? (ml[w][1][r] == 0.f ? 0.f : 1.f) : ex2(ml[w][0][r] - M);
            const float4 y = *reinterpret_cast<const float4*>(os + ((size_t)w * RT + r) * HD + d);
            L = fmaf(ml[w][1][r], f, L);
            x.x = fmaf(y.x, f, x.x), x.y = fmaf(y.y, f, x.y), x.z = fmaf(y.z, f, x.z), x.w = fmaf(y.w, f, x.w);
        }
        if (ns == 1) {
            const float inv = L == 0.f ? 0.f : 1.0f / L;
            const int row = row0 + r;
            store4(a.out.at((size_t)sq.r0 + row / a.G, h * a.G + row % a.G) + d, a.vec,
                   make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv));
        } else {
            float* y = part + (size_t)r * (HD + 2);
            *reinterpret_cast<float2*>(y + 2 + d) = make_float2(x.x, x.y);
            *reinterpret_cast<float2*>(y + 4 + d) = make_float2(x.z, x.w);
            if (d == 0) *reinterpret_cast<float2*>(y) = make_float2(M, L);
        }
    }
    if (ns == 1) return;
    // the split that arrives last joins them all, in their order
    __threadfence();
    __syncthreads();
    if (tid == 0) {
        last_cta = atomicAdd(p.tickets + item, 1u) == (uint32_t)ns - 1;
        if (last_cta) p.tickets[item] = 0;
    }
    __syncthreads();
    if (!last_cta) return;
    __threadfence();
    const float* all = p.part + item * p.splits * RT * (HD + 2);
    for (int i = tid; i < valid * (HD / 4); i += 32 * kStepWarps) {
        const int r = i / (HD / 4), d = 4 * (i % (HD / 4));
        float M = -INFINITY, L = 0.f;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int k = 0; k < ns; k++) {
            const float* y = all + ((size_t)k * RT + r) * (HD + 2);
            const float2 w = __ldcg(reinterpret_cast<const float2*>(y));
            const float2 u = __ldcg(reinterpret_cast<const float2*>(y + 2 + d)),
                         v = __ldcg(reinterpret_cast<const float2*>(y + 4 + d));
            const float to = fmaxf(M, w.x);
            const float fo = M == -INFINITY ? (L == 0.f ? 0.f : 1.f) : ex2(M - to),
                        fn = w.x == -INFINITY ? (w.y == 0.f ? 0.f : 1.f) : ex2(w.x - to);
            M = to;
            L = fmaf(L, fo, w.y * fn);
            x.x = fmaf(x.x, fo, u.x * fn), x.y = fmaf(x.y, fo, u.y * fn);
            x.z = fmaf(x.z, fo, v.x * fn), x.w = fmaf(x.w, fo, v.y * fn);
        }
        const float inv = L == 0.f ? 0.f : 1.0f / L;
        const int row = row0 + r;
        store4(a.out.at((size_t)sq.r0 + row / a.G, h * a.G + row % a.G) + d, a.vec,
               make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv));
    }
}

template <int HD, typename T>
cudaError_t launch_kv8_step(const Kv8Attn<T>& a, const Kv8StepPlan& p, cudaStream_t st) {
    const size_t smem = (size_t)kStepWarps * kStepStages * 32 * HD;
    const unsigned grid = (unsigned)(p.items * p.splits);
    static_assert(kStepStages * 32 >= 16 * 4, "the ring holds the warps' parts");
    auto go = [&](auto* kernel, std::atomic<uint32_t>& done) {
        const cudaError_t e = kv8_smem_once(kernel, (int)smem, p.device, done);
        if (e != cudaSuccess) return e;
        kernel<<<grid, 32 * kStepWarps, smem, st>>>(a, p);
        return cudaGetLastError();
    };
    if constexpr (sizeof(T) == 2) {
        static std::atomic<uint32_t> done16{0};
        if (!p.pair) return go(&kv8_attn_step_kernel<HD, T, false>, done16);
    }
    static std::atomic<uint32_t> done8{0};
    return go(&kv8_attn_step_kernel<HD, T, true>, done8);
}

#define POX_KV8_STEP(HD)                                                                                       \
    template cudaError_t launch_kv8_step<HD, float>(const Kv8Attn<float>&, const Kv8StepPlan&, cudaStream_t);   \
    template cudaError_t launch_kv8_step<HD, __half>(const Kv8Attn<__half>&, const Kv8StepPlan&, cudaStream_t); \
    template cudaError_t launch_kv8_step<HD, __nv_bfloat16>(const Kv8Attn<__nv_bfloat16>&, const Kv8StepPlan&,  \
                                                            cudaStream_t);
POX_KV8_STEP(32)
POX_KV8_STEP(64)
POX_KV8_STEP(128)

}  // namespace pox
