// kv8_prompt.cu -- attention of many rows (prompts and prompt chunks) over int8 pages on the 5th-generation
// tensor cores.
//
// The same mathematics as kv8_attn.cu: u_t = scale log2(e) a q . k_t + log2 b, p_t = 2^(u_t - m),
// out = sum p_t v_t / sum p_t / b with whole numbers k_t, v_t and page scales a, b. The rows of a kv head are its
// (token, query head of the group) pairs in order, 128 to a tile; causal masking is by each row's own position.
#include "kv8_attn.h"
#include "kv8_math.cuh"
#include "tc05.cuh"

namespace pox {

// D[tmem] (+)= A[tmem] * B[smem]^T: A is M = 128 lanes of packed f16 pairs, 8 columns for 16 k.
__device__ __forceinline__ void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                            uint32_t accumulate) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d_tmem),
        "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// eight operands of an asm statement, v[i] .. v[i + 7]
#define POX_V8(c, v, i) \
    c(v[i]), c(v[i + 1]), c(v[i + 2]), c(v[i + 3]), c(v[i + 4]), c(v[i + 5]), c(v[i + 6]), c(v[i + 7])
#define POX_R16 "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}"
#define POX_R32                                                    \
    "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"  \
    "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}"
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], " POX_R16 ";" ::POX_V8("r", r, 0), POX_V8("r", r, 8),
                 "r"(taddr)
                 : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float (&v)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 " POX_R16 ", [%16];"
                 : POX_V8("=f", v, 0), POX_V8("=f", v, 8)
                 : "r"(taddr)
                 : "memory");
    asm volatile("tcgen05.wait::ld.sync.aligned;" : POX_V8("+f", v, 0), POX_V8("+f", v, 8)::"memory");
}
// 32 columns of the warp's lanes, on their way; tmem_here(v) for each of them after tmem_wait_ld().
__device__ __forceinline__ void tmem_ask32(uint32_t taddr, float* v) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 " POX_R32 ", [%32];"
                 : POX_V8("=f", v, 0), POX_V8("=f", v, 8), POX_V8("=f", v, 16), POX_V8("=f", v, 24)
                 : "r"(taddr)
                 : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_here(float* v) {  // (no instruction: uses of v stay behind the wait)
    asm volatile("" : POX_V8("+f", v, 0), POX_V8("+f", v, 8), POX_V8("+f", v, 16), POX_V8("+f", v, 24));
}
__device__ __forceinline__ float4 lds_f4(uint32_t a) {
    const uint4 v = lds128(a);
    return make_float4(__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w));
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
template <int N>
__device__ __forceinline__ void regs_more() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_less() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

constexpr int kPromptKeys = 128;                   // tokens of a tile: 8 pages
constexpr int kPromptThreads = 512;                // two softmax warpgroups, the converters, the MMA warp's group
// registers of a thread of each group; the launch gives 128 to all, and these sum to as much
constexpr int kSoftmaxRegs = 184, kConvertRegs = 88, kMmaRegs = 56;
static_assert(2 * kSoftmaxRegs + kConvertRegs + kMmaRegs <= 4 * 128, "more registers than the launch has");

template <int HD>
struct PromptSmem {
    static constexpr int kQ = 128 * HD * 2;             // bytes of one q tile
    static constexpr int kHalf = kPromptKeys * HD * 2;  // K or V of a tile in f16
    static constexpr int kStages = 4;                   // two tiles of each
    static constexpr int total = 2 * kQ + kStages * kHalf;
};

// One CTA per (sequence, kv head, 256 rows): two tiles of 128 rows share every K and V tile. Warps 0-3 and 4-7
// hold the softmax of one tile each (a thread a row), warps 8-11 turn int8 pages into f16 operand tiles
// (exactly) in the 128-byte-swizzled K-major layout, one thread of warp 12 issues the products:
//   S = Q K^T (shared x shared -> TMEM), O += P V (P packed f16 in TMEM over S's columns, V shared).
// While one tile's softmax runs, the tensor core works on the other's products. The reference m of a row moves only when
// p would pass 2^8 (then its warp rescales O in TMEM), so that O is hardly ever read before the end. p is rounded to
// f16 (2^-11 of p, as f16 and bf16 outputs are rounded to no more), the sums of p and O are f32. f32 rows stay with the
// step kernel: carried as two f16 terms through these products, an output was 7e-6 off (the tensor core drops low bits
// as it adds up) where mma.sync is 3e-7 off.
// O stays in TMEM through the context, where each product cuts off what it adds to: 1.1e-9 of an output for each token
// seen, 1.3e-4 at 131072, below the roundings of f16 and of p.
// 8192 rows over themselves, 32 heads over 8 of 128, bf16: 657 to 670 us (632 on one box of six), 820 to 870 TFLOP/s, 50
// to 53 % of the measured rate of library products. The round trip of a tile bounds it: a row tile's next product waits
// for its softmax, and the two softmaxes together take longer than the products that they hide (tensor pipe 40 % busy,
// exponentials 41 %).
// An MMA completes in order with those issued before it: S of tile j ready means P V of tile j - 1 done.
template <int HD, typename T>
__global__ void __launch_bounds__(kPromptThreads, 1) kv8_attn_prompt_kernel(Kv8Attn<T> a, int min_rows) {
    using SM = PromptSmem<HD>;
    constexpr int NST = SM::kStages, QB = SM::kQ, HB = SM::kHalf;
    constexpr uint32_t TS = 0, TO = 256;  // TMEM columns: S of tile t at 128 t, O at 256 + HD t
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bars[2 * NST + 5];
    __shared__ float4 scal[2][8];  // of a tile's pages: a, log2 b, 1 / b
    __shared__ uint32_t tmem_base;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t smem = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t full = smem_u32(bars), empty = full + 8 * NST, sfull = empty + 8 * NST, pready = sfull + 16,
                   ofull = pready + 16;

    pdl_wait();
    pdl_launch_dependents();
    if (check_batch(a.b, a.err)) return;
    // Tile items of 256 rows: sequence s owns (row_starts[s] G + 255 s) / 256 .. (with room for its last, partial one).
    // Long tiles first: the last rows of a sequence see the most tokens.
    const uint32_t item = blockIdx.x / a.c.kvh, h = blockIdx.x - item * a.c.kvh;
    auto first_item = [&](uint32_t q) {
        return (uint32_t)(((unsigned long long)a.b.row_starts[q] * a.G + 255ull * q) / 256);
    };
    const uint32_t s = a.b.row_starts ? find_seq(a.b, item, first_item) : item;
    SeqSpan sq;
    if (!seq_span(a.b, s, sq, a.err)) return;
    const int rows = sq.n * a.G, k_tile = a.b.row_starts ? (int)(item - first_item(s)) : 0;
    const int row0 = ((rows + 255) / 256 - 1 - k_tile) * 256;
    if (rows < min_rows || k_tile < 0 || row0 < 0) return;
    // (what the outputs' addresses are made of waits in shared memory: in registers it made the softmax spill, 722 us
    // against 632)
    __shared__ uint32_t place_s[2];
    if (tid == 0) place_s[0] = row0, place_s[1] = sq.r0;
    const int pos0 = sq.ctx - sq.n, pmax = pos0 + (min(row0 + 256, rows) - 1) / a.G;
    const int nt = row0 + 128 < rows ? 2 : 1, nk = pmax < 0 ? 0 : pmax / kPromptKeys + 1;
    const int32_t* bt = a.b.btab + (size_t)s * a.b.mbps;
    const int last_page = pmax < 0 ? -1 : pmax / kPage;

    if (warp == 12) {
        if (lane == 0) {
            for (int i = 0; i < NST; i++) mbar_init(full + 8 * i, 4), mbar_init(empty + 8 * i, 1);
            for (int i = 0; i < 2; i++) mbar_init(sfull + 8 * i, 1), mbar_init(pready + 8 * i, 4);
            mbar_init(ofull, 1);
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        __syncwarp();
        tmem_alloc(smem_u32(&tmem_base), 512);
        tmem_relinquish();
    }
    const uint32_t qs = smem, kv = smem + 2 * QB;

    // q rows to f16 operand tiles (a thread a row), scaled by a power of two per row
    const int ti = warp >> 2, row = row0 + tid;  // softmax warps: the row of tile ti that this thread keeps
    const bool mine = tid < 256 && row < rows;
    float qf = 0.f;
    if (tid < 128 * nt) {
        const T* q = a.q.at((size_t)sq.r0 + (mine ? row / a.G : 0), h * a.G + (mine ? row % a.G : 0));
        float f = 1.f, inv = 1.f;
        if constexpr (!std::is_same<T, __half>::value) {
            float m = 0.f;
#pragma unroll 4
            for (int d = 0; d < HD; d += 4) {
                float v[4];
                load4(q + d, a.vec, v);
                m = fmaxf(fmaxf(m, fmaxf(fabsf(v[0]), fabsf(v[1]))), fmaxf(fabsf(v[2]), fabsf(v[3])));
            }
            f = row_factor(m, inv);
        }
        qf = inv * a.scale;
        const uint32_t r = tid & 127, qt = qs + ti * QB;
#pragma unroll 4
        for (int d = 0; d < HD; d += 8) {
            float v[8];
            load4(q + d, a.vec, *reinterpret_cast<float(*)[4]>(v));
            load4(q + d + 4, a.vec, *reinterpret_cast<float(*)[4]>(v + 4));
            uint32_t x[4];
#pragma unroll
            for (int i = 0; i < 4; i++) x[i] = mine ? pack_f16(v[2 * i] * f, v[2 * i + 1] * f) : 0u;
            sts128(qt + (d / 64) * (128 * 128) + sw128_off(r, (d % 64) / 8), x[0], x[1], x[2], x[3]);
        }
        fence_proxy_async_smem();
    }
    __syncthreads();
    tc_fence_after();
    const uint32_t tm = tmem_base;
    bool bad = false;

    if (warp < 8) {  // ---- softmax of tile ti
        regs_more<kSoftmaxRegs>();
        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16, ts = tm + TS + 128 * ti + lanes,
                       to = tm + TO + HD * ti + lanes;
        const int rpos = mine ? pos0 + row / a.G : 0x3fffffff;
        const int wpos = pos0 + (row0 + 32 * warp) / a.G;  // the first row of the warp sees no further
        float m = -INFINITY, ref = 0.f, l = 0.f;
        if (ti < nt) {
            for (int j = 0; j < nk; j++) {
                // the pages' scalars come with V (whose stage is free again only when this tile's p has been used)
                bad = __any_sync(0xffffffffu, !mbar_wait(full + 8 * ((2 * j + 1) % NST), ((2 * j + 1) / NST) & 1));
                if (!bad) bad = __any_sync(0xffffffffu, !mbar_wait(sfull + 8 * ti, j & 1));
                if (bad) break;
                tc_fence_after();
                // the tile's row in registers
                float x[kPromptKeys];
#pragma unroll
                for (int c = 0; c < 4; c++) tmem_ask32(ts + 32 * c, x + 32 * c);
                const uint32_t sc = smem_u32(scal[j & 1]);  // within a page u = S (qf a) + log2 b
                tmem_wait_ld();
#pragma unroll
                for (int c = 0; c < 4; c++) tmem_here(x + 32 * c);
                const int left = rpos - j * kPromptKeys;  // the last of the tile's tokens that the row sees
                auto softmax = [&](auto masked) {
                    constexpr bool CUT = decltype(masked)::value;
                    float mx = -INFINITY;
#pragma unroll
                    for (int g = 0; g < 8; g++) {
                        const float* y = x + 16 * g;
                        const float4 pg = lds_f4(sc + 16 * g);
                        const float f = qf * pg.x, pl = pg.y;
                        if (CUT) {
#pragma unroll
                            for (int i = 0; i < 16; i++)
                                mx = fmaxf(mx, 16 * g + i > left ? -INFINITY : fmaf(y[i], f, pl));
                        } else {
                            const float y0 = max3(y[0], y[1], y[2]), y1 = max3(y[3], y[4], y[5]),
                                        y2 = max3(y[6], y[7], y[8]), y3 = max3(y[9], y[10], y[11]),
                                        y4 = max3(y[12], y[13], y[14]);
                            mx = fmaxf(mx, fmaf(fmaxf(max3(y0, y1, y2), max3(y3, y4, y[15])), f, pl));
                        }
                    }
                    if (__any_sync(0xffffffffu, mx > m + 8.0f)) {
                        const float go = mx > m + 8.0f ? mx : m;
                        const float d = m == -INFINITY ? (go == -INFINITY ? 1.f : 0.f) : ex2(m - go);
                        m = go, ref = go == -INFINITY ? 0.f : go;
                        l *= d;
                        if (j) {
#pragma unroll
                            for (int c = 0; c < HD / 16; c++) {
                                float y[16];
                                tmem_ld16(to + 16 * c, y);
#pragma unroll
                                for (int i = 0; i < 16; i++) y[i] *= d;
                                tmem_st16(to + 16 * c, reinterpret_cast<const uint32_t(&)[16]>(y));
                            }
                        }
                    }
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        uint32_t hi[16];
#pragma unroll
                        for (int g = 2 * c; g < 2 * c + 2; g++) {
                            const float4 pg = lds_f4(sc + 16 * g);
                            const float f = qf * pg.x, off = pg.y - ref;
                            const uint64_t f2 = pair2(f, f), off2 = pair2(off, off);
                            uint64_t sum2 = 0;
#pragma unroll
                            for (int i = 0; i < 16; i += 2) {
                                float2 z = both(fma2(pair2(x[16 * g + i], x[16 * g + i + 1]), f2, off2));
                                if (CUT) {
                                    if (16 * g + i > left) z.x = -INFINITY;
                                    if (16 * g + i + 1 > left) z.y = -INFINITY;
                                }
                                z.x = ex2(z.x), z.y = ex2(z.y);
                                sum2 = add2(sum2, pair2(z.x, z.y));
                                hi[8 * (g & 1) + i / 2] = pack_f16(z.x, z.y);
                            }
                            const float sum = both(sum2).x + both(sum2).y;
                            if (!CUT || sum != 0.f) l = fmaf(sum, pg.z, l);  // (an unseen page's scale may be anything)
                        }
                        tmem_st16(ts + 16 * c, hi);  // over columns of S
                    }
                };
                if (j * kPromptKeys + kPromptKeys - 1 > wpos) softmax(std::true_type());
                else softmax(std::false_type());
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(pready + 8 * ti);
            }
            if (nk && !bad) bad = __any_sync(0xffffffffu, !mbar_wait(ofull, 0));
            tc_fence_after();
            const float inv = l == 0.f ? 0.f : 1.0f / l;
            const volatile uint32_t* place = place_s;
            const int last_row = (int)place[0] + tid;
            T* y = a.out.at((size_t)place[1] + (mine ? last_row / a.G : 0), h * a.G + (mine ? last_row % a.G : 0));
#pragma unroll
            for (int c = 0; c < HD / 32; c++) {
                float x[32];
                if (nk) tmem_ld32(to + 32 * c, x);
                else
#pragma unroll
                    for (int i = 0; i < 32; i++) x[i] = 0.f;
                if (mine && !bad)
#pragma unroll
                    for (int i = 0; i < 32; i += 4)
                        store4(y + 32 * c + i, a.vec,
                               make_float4(x[i] * inv, x[i + 1] * inv, x[i + 2] * inv, x[i + 3] * inv));
            }
        }
    } else if (warp < 12) {  // ---- converters: pages 2 w and 2 w + 1 of each tile
        regs_less<kConvertRegs>();
        const int w = warp - 8, b = lane & 7, g = lane >> 3;
        constexpr int NI = HD / 16;  // 16-byte pieces of K (or V) per lane and tile
        uint4 r[NI];  // K's pieces, then V's: the warps run ahead of the products, and more registers are the softmax's
        // lane i looks after page i % 2 of the warp's two: its entry asked for two tiles ahead, its scales one
        // (loads that every lane makes, looked at a tile later: behind a branch each tile began with their latency)
        auto entry = [&](int j) { return bt[min(8 * j + 2 * w + (lane & 1), max(last_page, 0))]; };
        auto there = [&](int blk, int j) {
            const bool in = 8 * j + 2 * w + (lane & 1) <= last_page;
            const bool ok = in && blk >= 0 && (uint32_t)blk < a.c.num_blocks;
            if (in && !ok && lane < 2) atomicOr(a.err, kErrAttnPage);
            return ok;
        };
        auto scales = [&](int blk, bool ok) {
            return *reinterpret_cast<const float2*>(a.c.scales + ((size_t)(ok ? blk : 0) * a.c.kvh + h) * 2);
        };
        // (a page that is left out, or past the context, has p = 0: block 0 stands in for it, any bytes do)
        auto page_of = [&](int blk, bool ok, int i) {
            return a.c.pages + ((size_t)__shfl_sync(0xffffffffu, ok ? blk : 0, i) * a.c.kvh + h) * (32 * HD);
        };
        auto load_k = [&](const int8_t* p0, const int8_t* p1) {
#pragma unroll
            for (int i = 0; i < NI; i++) {
                const int8_t* p = i < NI / 2 ? p0 : p1;
                const int q = i % (NI / 2), t = 8 * (q & 1) + b, c = 4 * (q >> 1) + g;
                r[i] = ldg128_nc(p + kv8_k_off<HD>(t, 16 * c));
            }
        };
        auto load_v = [&](const int8_t* p0, const int8_t* p1) {
#pragma unroll
            for (int i = 0; i < NI; i++) {
                const int8_t* p = i < NI / 2 ? p0 : p1;
                r[i] = ldg128_nc(p + kv8_v_off<HD>(0, 32 * (i % (NI / 2)) + 8 * g + b));
            }
        };
        auto put = [&](uint32_t at0, uint32_t at1, uint4 x) {
            uint32_t f[8];
            i8x4_to_f16x4(x.x, f[0], f[1]);
            i8x4_to_f16x4(x.y, f[2], f[3]);
            i8x4_to_f16x4(x.z, f[4], f[5]);
            i8x4_to_f16x4(x.w, f[6], f[7]);
            sts128(at0, f[0], f[1], f[2], f[3]);
            sts128(at1, f[4], f[5], f[6], f[7]);
        };
        auto ready = [&](int st) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(full + 8 * st);
        };
        int blk = nk ? entry(0) : 0, next = nk ? entry(1) : 0;
        bool ok = there(blk, 0);
        float2 ab = scales(blk, ok);
        const int8_t *p0 = page_of(blk, ok, 0), *p1 = page_of(blk, ok, 1);
        if (nk) load_k(p0, p1);
        for (int j = 0; j < nk; j++) {
            // a page that is left out: u is -inf whatever S
            const float b0 = fmaxf(ab.y, 1e-30f);
            const float4 sc = ok ? make_float4(ab.x, log2f(b0 + (ab.y - ab.y)), 1.0f / b0, 0.f)
                                 : make_float4(0.f, -INFINITY, 0.f, 0.f);
            blk = next, next = entry(j + 2);
            ok = there(blk, j + 1);
            ab = scales(blk, ok);
            int n = 2 * j, st = n % NST;
            if (n >= NST) bad = __any_sync(0xffffffffu, !mbar_wait(empty + 8 * st, (n / NST - 1) & 1));
            if (bad) break;
#pragma unroll
            for (int i = 0; i < NI; i++) {
                const int q = i % (NI / 2), t = 16 * (2 * w + i / (NI / 2)) + 8 * (q & 1) + b, c = 4 * (q >> 1) + g;
                const uint32_t base = kv + st * HB + (c / 4) * (kPromptKeys * 128);
                put(base + sw128_off(t, 2 * (c % 4)), base + sw128_off(t, 2 * (c % 4) + 1), r[i]);
            }
            ready(st);
            load_v(p0, p1);
            n++, st = n % NST;
            if (n >= NST) bad = __any_sync(0xffffffffu, !mbar_wait(empty + 8 * st, (n / NST - 1) & 1));
            if (bad) break;
            if (lane < 2) scal[j & 1][2 * w + lane] = sc;
#pragma unroll
            for (int i = 0; i < NI; i++) {
                const int page = 2 * w + i / (NI / 2), d = 32 * (i % (NI / 2)) + 8 * g + b;
                const uint32_t base = kv + st * HB + (page / 4) * (HD * 128);
                put(base + sw128_off(d, 2 * (page % 4)), base + sw128_off(d, 2 * (page % 4) + 1), r[i]);
            }
            ready(st);
            p0 = page_of(blk, ok, 0), p1 = page_of(blk, ok, 1);
            if (j + 1 < nk) load_k(p0, p1);
        }
    } else {  // ---- the products: one thread of warp 12
        regs_less<kMmaRegs>();
        if (warp == 12 && lane == 0 && nk) {
            constexpr uint32_t is = umma_idesc_f16(128, kPromptKeys), ip = umma_idesc_f16(128, HD);
            auto wait_full = [&](int n) {
                if (!bad) bad = !mbar_wait(full + 8 * (n % NST), (n / NST) & 1);
                tc_fence_after();
            };
            auto release = [&](int n) {  // the stage, if the converters wait for it (nothing arrives there after the end)
                if (n + NST < 2 * nk) umma_commit(empty + 8 * (n % NST));
            };
            auto scores = [&](int t, int j) {
                const uint32_t k0 = kv + (2 * j % NST) * HB;
#pragma unroll
                for (int k = 0; k < HD / 16; k++)
                    umma_f16(tm + TS + 128 * t, umma_desc_sw128(qs + t * QB + (k / 4) * (128 * 128)) + 2 * (k % 4),
                             umma_desc_sw128(k0 + (k / 4) * (kPromptKeys * 128)) + 2 * (k % 4), is, k);
                umma_commit(sfull + 8 * t);
            };
            auto values = [&](int t, int j) {
                if (!bad) bad = !mbar_wait(pready + 8 * t, j & 1);
                tc_fence_after();
                if (bad) return;
                const uint32_t v0 = kv + ((2 * j + 1) % NST) * HB;
#pragma unroll
                for (int k = 0; k < kPromptKeys / 16; k++)
                    umma_f16_ts(tm + TO + HD * t, tm + TS + 128 * t + 8 * k,
                                umma_desc_sw128(v0 + (k / 4) * (HD * 128)) + 2 * (k % 4), ip, j || k);
            };
            wait_full(0);
            if (!bad) {
                for (int t = 0; t < nt; t++) scores(t, 0);
                release(0);
            }
            for (int j = 0; j < nk && !bad; j++) {
                wait_full(2 * j + 1);
                for (int t = 0; t < nt && !bad; t++) {
                    values(t, j);
                    if (t == nt - 1) release(2 * j + 1);
                    if (j + 1 < nk) {
                        if (t == 0) wait_full(2 * j + 2);
                        if (!bad) scores(t, j + 1);
                        if (t == nt - 1) release(2 * j + 2);
                    }
                }
            }
            umma_commit(ofull);
            if (bad) mbar_wait(ofull, 0);  // what was issued ends before the tensor memory is given back
        }
    }
    if (bad && lane == 0) atomicOr(a.err, kErrWaitRing);
    tc_fence_before();
    __syncthreads();
    if (warp == 12) {
        tc_fence_after();
        tmem_dealloc(tm, 512);
    }
}

template <int HD, typename T>
cudaError_t launch_kv8_prompt(const Kv8Attn<T>& a, int min_rows, int device, cudaStream_t st) {
    constexpr int smem = PromptSmem<HD>::total + 1024;
    static_assert(smem + 1024 <= 227 * 1024, "shared memory of a CTA");
    static std::atomic<uint32_t> done{0};
    const cudaError_t e = kv8_smem_once(&kv8_attn_prompt_kernel<HD, T>, smem, device, done);
    if (e != cudaSuccess) return e;
    return launch_pdl(kv8_attn_prompt_kernel<HD, T>, dim3((unsigned)kv8_prompt_grid(a.b, a.c.kvh, a.G)),
                      dim3(kPromptThreads), smem, st, a, min_rows);
}

#define POX_KV8_PROMPT(HD)                                                                                  \
    template cudaError_t launch_kv8_prompt<HD, __half>(const Kv8Attn<__half>&, int, int, cudaStream_t);     \
    template cudaError_t launch_kv8_prompt<HD, __nv_bfloat16>(const Kv8Attn<__nv_bfloat16>&, int, int, cudaStream_t);
POX_KV8_PROMPT(64)
POX_KV8_PROMPT(128)

}  // namespace pox
