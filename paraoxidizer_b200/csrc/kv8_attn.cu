// kv8_attn.cu -- attention of few rows over int8 pages with one scale per page, kv head and side.
//
// For row r (a query head at a token) of one kv head, with page scales a (of k) and b (of v):
//   s_t = scale log2(e) a q . k_t,   u_t = s_t + log2 b,   p_t = 2^(u_t - m),   m about max u_t
//   out = sum_t p_t v_t / sum_t p_t / b
// where k_t and v_t are the stored whole numbers. Taking the maximum over u instead of s puts the scale of
// v into the exponent: the products see whole numbers and p <= 2^8, and no page's scale multiplies a tile.
#include "kv8_attn.h"
#include "kv8_math.cuh"
#include "tc05.cuh"

namespace pox {

// The ring of a warp: stages of two pages. Three CTAs to an SM at 128 dims, four below (registers and shared memory).
template <int HD>
struct StepRing {
    static constexpr int kPageBytes = 32 * HD, kPairBytes = 2 * kPageBytes, kStages = HD == 128 ? 2 : 3;
};

// Two f16 from the low (high) two bytes of a word of int8.
//   EXACT: the whole numbers q themselves.
//   else:  (q + 128) 2^-24, the byte with its sign bit flipped as a subnormal f16: three instructions a word instead
//          of five; a product is then off by 128 2^-24 times the sum of the other operand, which it starts below zero
//          by. For sums over a head's dims only: along a context the offset grows past what it hides (at 131072 tokens of
//          diffuse scores an output was 14 % off), so V enters exactly.
template <bool EXACT>
__device__ __forceinline__ void bytes_to_f16(uint32_t v, uint32_t& r0, uint32_t& r1) {
    if constexpr (EXACT) {
        i8x4_to_f16x4(v, r0, r1);
    } else {
        const uint32_t u = v ^ 0x80808080u;
        r0 = prmt(u, 0u, 0x4140u);
        r1 = prmt(u, 0u, 0x4342u);
    }
}
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {  // an 8 x 8 matrix of f16 pairs across the warp
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
// D = A B + (c0, c1, c0, c1)
__device__ __forceinline__ void mma_start(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1, float c0, float c1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%10,%11};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1));
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
    uint32_t r;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(r) : "r"(a));
    return r;
}

// The work of a launch is a line of units: for each sequence in turn, for each kv head and tile of 8 NT rows,
// kItemUnits for starting on it and one for each page of the sequence. Every CTA takes an equal run of the line,
// whatever the lengths are (with a CTA per split of the longest context, 122 us against 106 at three sequences of 131k,
// 109k and 61k tokens: a quarter of the SMs' time went by idle). A long item that a run's
// end cuts leaves its part in the CTA's place (0: of an item begun before, 1: of one that goes on), and the CTA that
// comes last joins them in order.
//
// Within an item each warp streams whole pages (K and V of 16 tokens of the kv head, 32 HD contiguous bytes) through a
// ring of its own with one bulk copy a page, two pages a turn, and runs both products transposed on mma.sync m16n8k16
// with f32 accumulators, so that a page is the 16 rows of A and 8 query rows fill N:
//   S^T (tokens x rows) = K Q^T,   O^T (dims x rows) = V^T P^T.
// The MMA does not care in which order k and the rows of A run, so they run as the page's bytes lie: lane (g, t) takes
// 16 dims of the tokens 4 (g / 2) + g % 2 (+ 2) for the first product and the four tokens 4 t .. 4 t + 3 of a dim for
// the second, and P^T is S^T's own fragment, transposed in registers.
// f32 rows: q and p as two f16 terms each (22 bits), bytes converted exactly. 16-bit rows: q exact, K's bytes with the
// offset of bytes_to_f16, V's exactly; p two terms for f16 outputs of up to 8 rows (so that only the output's own
// rounding remains), one for bf16 and for more rows (2^-11 of p).
//
// What bounds it: HBM where the contexts are long (64 sequences of 3800 to 4400 tokens, 64 heads over 8 of 128, bf16:
// 541 MB in 97 us, 85 % of the measured copy rate; the three above 109 us, 81 %); the start and joining of items
// where there are many short ones (37 sequences of up to 2011 tokens, 12 heads of 64: 25 us, its bytes 8.4); for f32
// rows the products of two terms each (20 prompts of up to 257 rows, 14 heads over 2 of 64: 128 us, mma.sync pipe 40 %
// and issue slots 45 % busy at the 8 warps that the registers leave an SM); one sequence of 640 tokens the launch (5.6).
constexpr uint32_t kWholePages = 128;

template <int HD, typename T, int NT>
__global__ void __launch_bounds__(32 * kStepWarps, NT == 1 ? (HD == 128 ? 3 : 4) : 2)
    kv8_attn_step_kernel(Kv8Attn<T> a, Kv8StepPlan p) {
    constexpr bool F32 = sizeof(T) == 4, PLO = F32 || (std::is_same<T, __half>::value && NT == 1);
    constexpr int RT = 8 * NT, KW = HD / 16, NJ = HD / 16, NST = StepRing<HD>::kStages;
    constexpr int PB = StepRing<HD>::kPageBytes, SB = StepRing<HD>::kPairBytes;
    constexpr float kOffset = 128.0f / 16777216.0f;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ __align__(8) uint64_t bars[kStepWarps][NST];
    __shared__ float ml[kStepWarps][2][RT];
    __shared__ uint32_t last_cta;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const uint32_t ring = smem_u32(smem) + warp * NST * SB, bar = smem_u32(&bars[warp][0]);
    if (lane == 0) {
        for (int i = 0; i < NST; i++) mbar_init(bar + 8 * i, 2);  // the lanes of its two pages
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    pdl_wait();
    pdl_launch_dependents();
    // units of a sequence (one item at least, so that rows that see nothing are written), and where this CTA's run begins
    auto units = [&](uint32_t s, SeqSpan& q) -> unsigned long long {
        if (s >= a.b.seqs || !seq_span(a.b, s, q, a.err)) return 0;
        const int rows = q.n * a.G;
        if (rows > p.most_rows) return 0;
        return (unsigned long long)a.c.kvh * ((rows + RT - 1) / RT) * (kItemUnits + max((q.ctx + kPage - 1) / kPage, 1));
    };
    SeqSpan sq;
    const unsigned long long mine = units(lane, sq);
    unsigned long long all_units = mine;
    for (uint32_t s0 = 32; s0 < a.b.seqs; s0 += 32) {
        SeqSpan q;
        all_units += units(s0 + lane, q);
    }
#pragma unroll
    for (int k = 16; k; k >>= 1) all_units += __shfl_xor_sync(0xffffffffu, all_units, k);
    if (all_units >= 0xff000000u) {
        if (tid == 0) atomicOr(a.err, kErrBatch);
        return;
    }
    const uint32_t total = (uint32_t)all_units, run = max((total + gridDim.x - 1) / gridDim.x, (uint32_t)p.min_units);
    // An item of up to `whole` pages is not cut (joining costs about what 64 pages do), and none within `edge` of its
    // ends: the border goes to the nearer end.
    const uint32_t whole = min(kWholePages, 2 * run), edge = min(16u, run / 2);
    auto border = [&](uint32_t u, uint32_t all) {  // a border u units into an item of `all`
        if (all - kItemUnits <= whole) return 2 * u < all ? 0u : all;
        return u < kItemUnits + edge ? 0u : u > all - edge ? all : u;
    };
    if ((unsigned long long)run * blockIdx.x >= total) return;
    const uint32_t x_begin = run * blockIdx.x, x_end = min(total - x_begin, run) + x_begin;
    uint32_t s = 0, base = 0;  // the sequence that holds x_begin, and the line's place where it begins
    for (uint32_t s0 = 0;; s0 += 32) {
        if (s0 >= a.b.seqs) {  // (lengths that change while the kernel runs: no loop depends on them)
            if (tid == 0) atomicOr(a.err, kErrBatch);
            return;
        }
        SeqSpan q;
        const uint32_t u = s0 ? (uint32_t)units(s0 + lane, q) : (uint32_t)mine;
        uint32_t sum = u;
#pragma unroll
        for (int k = 1; k < 32; k *= 2) {
            const uint32_t y = __shfl_up_sync(0xffffffffu, sum, k);
            if (lane >= k) sum += y;
        }
        const unsigned m = __ballot_sync(0xffffffffu, base + sum > x_begin);
        if (m) {
            s = s0 + __ffs(m) - 1;
            base += __shfl_sync(0xffffffffu, sum - u, __ffs(m) - 1);
            break;
        }
        base += __shfl_sync(0xffffffffu, sum, 31);
    }

    bool bad = false;
    int st = 0, ph = 0;
    uint32_t su = (uint32_t)units(s, sq), all = kItemUnits + max((sq.ctx + kPage - 1) / kPage, 1);
    uint32_t item = (x_begin - base) / all;
    uint32_t u0 = border(x_begin - base - item * all, all);  // of the item, this CTA's first unit
    for (;; item++, u0 = 0) {  // the items of this CTA's run
        uint32_t x0 = base + item * all;  // where the item begins
        while (x0 - base >= su) {  // the sequence is done
            base += su;
            if (base >= x_end || ++s >= a.b.seqs) return;
            su = (uint32_t)units(s, sq);
            all = kItemUnits + max((sq.ctx + kPage - 1) / kPage, 1);
            item = 0, x0 = base;
        }
        if (x0 >= x_end) return;
        const uint32_t u1 = all <= x_end - x0 ? all : border(x_end - x0, all);
        if (u0 >= u1) continue;
        const int rows = sq.n * a.G, tiles = (rows + RT - 1) / RT;
        auto token = [&](int row) { return sq.n == 1 ? 0 : row / a.G; };  // of a valid row
        // tiles of a sequence in the order first, last, second, ..: early ones see fewer pages of a chunk
        const int h = tiles == 1 ? (int)item : item / tiles, k_rt = item - h * tiles;
        const int row0 = (k_rt & 1 ? tiles - 1 - k_rt / 2 : k_rt / 2) * RT;
        const int pos0 = sq.ctx - sq.n, pmin = pos0 + token(row0), pmax = pos0 + token(min(row0 + RT, rows) - 1);
        const int pages = pmax < 0 ? 0 : pmax / kPage + 1;
        const int page0 = max((int)u0 - kItemUnits, 0), page1 = min(pages, (int)u1 - kItemUnits);
        // the CTA that holds the item's first part, and the parts: one more than the borders that cut it
        uint32_t c0 = blockIdx.x, ns = 1;
        if (u0 > 0 || u1 < all) {
            const uint32_t i0 = (x0 + kItemUnits + edge + run - 1) / run, i1 = (x0 + all - edge) / run;
            c0 = i0 - 1, ns = i1 - i0 + 2;
        }

        // the rows: lane (g, t) the dims of row g that t takes of a token (asked for before anything queues up behind
        // the pages)
        float qv[NT][KW][4];
#pragma unroll
        for (int n = 0; n < NT; n++) {
            const int row = row0 + 8 * n + g;
            const bool ok = row < rows;
            const int tk = ok ? token(row) : 0;
            const T* q = a.q.at((size_t)sq.r0 + tk, h * a.G + (ok ? row - tk * a.G : 0));
#pragma unroll
            for (int w = 0; w < KW; w++) {
                const int d = HD == 32 ? 8 * t + 4 * w : 64 * (w / 4) + 16 * t + 4 * (w % 4);
                if (ok) load4(q + d, a.vec, qv[n][w]);
                else qv[n][w][0] = qv[n][w][1] = qv[n][w][2] = qv[n][w][3] = 0.f;
            }
        }

        // this warp's pages: first, first + W, ..; lane i looks after the i-th of 32, and of the next 32: their
        // entries are asked for 32 pages ahead, their scales when the entries are there
        const int first = page0 + warp, cnt = first < page1 && !bad ? (page1 - first + kStepWarps - 1) / kStepWarps : 0;
        struct Entry {
            const int8_t* page;  // (one out of range: page 0, unread)
            float2 ab;
            unsigned there;
        } cur, nxt;
        auto entry = [&](int i) { return i < cnt ? a.b.btab[(size_t)s * a.b.mbps + first + i * kStepWarps] : 0; };
        auto resolve = [&](int blk, int i) {
            Entry e{nullptr, make_float2(0.f, 0.f), 0};
            const bool there = i < cnt && blk >= 0 && (uint32_t)blk < a.c.num_blocks;
            if (i < cnt) {
                if (!there) atomicOr(a.err, kErrAttnPage);
                const size_t place = there ? (size_t)blk * a.c.kvh + h : 0;
                e.page = a.c.pages + place * PB;
                e.ab = *reinterpret_cast<const float2*>(a.c.scales + place * 2);
            }
            e.there = __ballot_sync(0xffffffffu, there);
            return e;
        };
        // log2 b; a scale of 0 stands for zeros whatever the bytes: 1e-30 of them is nothing next to any other page
        float lb, ib;
        auto logs = [&](const Entry& e) {
            lb = log2f(fmaxf(e.ab.y, 1e-30f) + (e.ab.y - e.ab.y)), ib = 1.0f / fmaxf(e.ab.y, 1e-30f);
        };
        // pages i and i + 1 of this warp into a stage, by the lanes that look after them
        auto fetch = [&](const int8_t* page, int i, int st) {
            const uint32_t k = lane - (i & 31);
            if (k < 2) {
                if (i + (int)k < cnt) {
                    mbar_expect_tx(bar + 8 * st, PB);
                    bulk_g2s(ring + st * SB + k * PB, page, PB, bar + 8 * st);
                } else {
                    mbar_arrive(bar + 8 * st);
                }
            }
        };
        cur = resolve(entry(lane), lane);
        for (int i = 0, k = st; i < min(cnt, 2 * NST); i += 2) {
            fetch(cur.page, i, k);
            if (++k == NST) k = 0;
        }
        int ahead = entry(32 + lane);
        logs(cur);

        // B fragments of the rows. Then, for the rows 2 t and 2 t + 1 that this lane's scores belong to: what takes a
        // product to a score, its offset, and the last position seen
        uint32_t qb[NT][F32 ? 2 : 1][KW][2];
        float qf[NT][2], qo[NT][2];
        int rpos[NT][2];
#pragma unroll
        for (int n = 0; n < NT; n++) {
            float f = 1.f, inv = 1.f, sum = 0.f;
            if constexpr (!std::is_same<T, __half>::value) {
                float m = 0.f;
#pragma unroll
                for (int w = 0; w < KW; w++)
#pragma unroll
                    for (int i = 0; i < 4; i++) m = fmaxf(m, fabsf(qv[n][w][i]));
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
                f = row_factor(m, inv);
            }
#pragma unroll
            for (int w = 0; w < KW; w++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const float x = qv[n][w][2 * i] * f, y = qv[n][w][2 * i + 1] * f;
                    qb[n][0][w][i] = pack_f16(x, y);
                    if constexpr (F32) {
                        const float2 hi = unpack_f16(qb[n][0][w][i]);
                        qb[n][F32][w][i] = pack_f16(x - hi.x, y - hi.y);
                    } else {
                        sum += x + y;  // (16-bit rows are f16 exactly)
                    }
                }
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
#pragma unroll
            for (int e = 0; e < 2; e++) {
                qf[n][e] = __shfl_sync(0xffffffffu, inv, 8 * t + 4 * e) * a.scale * (F32 ? 1.0f : 16777216.0f);
                qo[n][e] = F32 ? 0.f : -kOffset * __shfl_sync(0xffffffffu, sum, 8 * t + 4 * e);
                const int r = row0 + 8 * n + 2 * t + e;
                rpos[n][e] = r < rows ? pos0 + token(r) : 0;
            }
        }

        // m: the reference (-inf until a row has seen something); ref: m, or 0
        float o[NT][NJ][4], m[NT][2], ref[NT][2], l[NT][2];
#pragma unroll
        for (int n = 0; n < NT; n++) {
#pragma unroll
            for (int j = 0; j < NJ; j++) o[n][j][0] = o[n][j][1] = o[n][j][2] = o[n][j][3] = 0.f;
#pragma unroll
            for (int e = 0; e < 2; e++) m[n][e] = -INFINITY, ref[n][e] = 0.f, l[n][e] = 0.f;
        }
        const int tok = 4 * (g >> 1) + (g & 1);
        const uint32_t k_at = HD == 32 ? tok * HD + 8 * t : tok * HD + 16 * t, swap = HD == 128 ? (g & 1) << 6 : 0,
                       v_at = kPage * HD + g * kPage + 4 * t;
        for (int i = 0; i < cnt; i += 2) {
            if ((i & 31) == 8) nxt = resolve(ahead, (i & ~31) + 32 + lane);
            if ((i & 31) == 0 && i) {
                cur = nxt, logs(cur);
                ahead = entry(i + 32 + lane);
            }
            const uint32_t at = ring + st * SB;
            bad = __any_sync(0xffffffffu, !mbar_wait(bar + 8 * st, ph));
            const int page = first + i * kStepWarps;
            const bool open = (cur.there >> (i & 31) & 3) == 3 && (page + kStepWarps + 1) * kPage - 1 <= pmin;
            float u[2][NT][4], pi[2];
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const uint32_t kb = at + k * PB + k_at;
                const float pa = __shfl_sync(0xffffffffu, cur.ab.x, (i & 31) + k),
                            pl = __shfl_sync(0xffffffffu, lb, (i & 31) + k);
                pi[k] = __shfl_sync(0xffffffffu, ib, (i & 31) + k);
                // S^T: tokens tok (rows g of A) and tok + 2 (rows g + 8)
                uint32_t kw[2][KW];
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    if constexpr (HD == 32) {
                        const uint2 x = lds64(kb + 2 * r * HD);
                        kw[r][0] = x.x, kw[r][1] = x.y;
                    } else {
#pragma unroll
                        for (int c = 0; c < HD / 64; c++) {
                            const uint4 x = lds128(kb + 2 * r * HD + (c ? 64 - swap : swap));
                            kw[r][4 * c] = x.x, kw[r][4 * c + 1] = x.y, kw[r][4 * c + 2] = x.z, kw[r][4 * c + 3] = x.w;
                        }
                    }
                }
                float low[F32 ? NT : 1][4];  // f32 rows: the second terms by themselves (see the other product)
#pragma unroll
                for (int w = 0; w < KW; w++) {
                    uint32_t a0, a1, a2, a3;
                    bytes_to_f16<F32>(kw[0][w], a0, a2);
                    bytes_to_f16<F32>(kw[1][w], a1, a3);
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        if (w == 0)
                            mma_start(u[k][n], a0, a1, a2, a3, qb[n][0][w][0], qb[n][0][w][1], qo[n][0], qo[n][1]);
                        else mma_16816(u[k][n], a0, a1, a2, a3, qb[n][0][w][0], qb[n][0][w][1]);
                        if constexpr (F32) {
                            if (w == 0) mma_start(low[n], a0, a1, a2, a3, qb[n][F32][w][0], qb[n][F32][w][1], 0.f, 0.f);
                            else mma_16816(low[n], a0, a1, a2, a3, qb[n][F32][w][0], qb[n][F32][w][1]);
                        }
                    }
                }
                // u of tokens tok, tok + 2 and rows 2 t, 2 t + 1
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        if constexpr (F32) u[k][n][e] += low[n][e];
                        u[k][n][e] = fmaf(u[k][n][e], qf[n][e & 1] * pa, pl);
                    }
            }
            if (!open) {
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    const bool seen = cur.there >> ((i & 31) + k) & 1;
#pragma unroll
                    for (int n = 0; n < NT; n++)
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            if (!seen || (page + k * kStepWarps) * kPage + tok + 2 * (e >> 1) > rpos[n][e & 1])
                                u[k][n][e] = -INFINITY;
                }
            }
            bool grow = false;
            float mx[NT][2];
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    mx[n][e] = fmaxf(fmaxf(u[0][n][e], u[0][n][2 + e]), fmaxf(u[1][n][e], u[1][n][2 + e]));
                    grow |= mx[n][e] > m[n][e] + 8.0f;
                }
            // the reference moves only when p would pass 2^8: after the first pages it hardly ever does
            if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        float to = mx[n][e];
#pragma unroll
                        for (int k = 4; k < 32; k *= 2) to = fmaxf(to, __shfl_xor_sync(0xffffffffu, to, k));
                        to = to > m[n][e] + 8.0f ? to : m[n][e];
                        const float f = m[n][e] == -INFINITY ? (to == -INFINITY ? 1.f : 0.f) : ex2(m[n][e] - to);
                        m[n][e] = to, ref[n][e] = to == -INFINITY ? 0.f : to;
                        l[n][e] *= f;
#pragma unroll
                        for (int j = 0; j < NJ; j++) o[n][j][e] *= f, o[n][j][2 + e] *= f;
                    }
            }
            uint32_t pb[2][NT][PLO ? 2 : 1][2];  // B fragments of P^T: tokens 4 t, 4 t + 1 | 4 t + 2, 4 t + 3 of row g
#pragma unroll
            for (int k = 0; k < 2; k++)
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    float x[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) x[e] = ex2(u[k][n][e] - ref[n][e & 1]);
#pragma unroll
                    for (int r = 0; r < 2; r++) {
                        const uint32_t hi = pack_f16(x[2 * r], x[2 * r + 1]);
                        pb[k][n][0][r] = transpose8(hi);
                        if constexpr (PLO) {
                            const float2 z = unpack_f16(hi);
                            pb[k][n][PLO][r] = transpose8(pack_f16(x[2 * r] - z.x, x[2 * r + 1] - z.y));
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        // (p in f32: a page's p may be nothing in f16 next to its part of l. An unseen page's scale may
                        // be anything.)
                        const float y = x[e] + x[2 + e];
                        if (open || y != 0.f) l[n][e] = fmaf(y, pi[k], l[n][e]);
                    }
                }
            // The pages' products by themselves, then added to o: the tensor core cuts off what it adds up, and chained
            // through, contexts of thousands of tokens were 2.0e-6 off in f32 (now, with the second terms of the scores
            // apart as well, 0.5e-6).
#pragma unroll
            for (int j = 0; j < NJ; j++) {
                float z[NT][4];
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    uint32_t a0, a1, a2, a3;
                    const uint32_t vb = at + k * PB + v_at + 16 * j * kPage;
                    bytes_to_f16<true>(lds32(vb), a0, a2);
                    bytes_to_f16<true>(lds32(vb + 8 * kPage), a1, a3);
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        if (k == 0) mma_start(z[n], a0, a1, a2, a3, pb[k][n][0][0], pb[k][n][0][1], 0.f, 0.f);
                        else mma_16816(z[n], a0, a1, a2, a3, pb[k][n][0][0], pb[k][n][0][1]);
                        if constexpr (PLO) mma_16816(z[n], a0, a1, a2, a3, pb[k][n][PLO][0], pb[k][n][PLO][1]);
                    }
                }
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int e = 0; e < 4; e++) o[n][j][e] += z[n][e];
            }
            __syncwarp();  // every lane has read the stage
            if (bad) {  // a copy did not come in time: give the ones in flight as long again, and leave
                for (int k = i; k < min(cnt, i + 2 * NST); k += 2) {
                    mbar_wait(bar + 8 * st, ph);
                    if (++st == NST) st = 0, ph ^= 1;
                }
                if (lane == 0) atomicOr(a.err, kErrWaitRing);
                break;
            }
            const int to = i + 2 * NST;
            if (to < cnt) fetch((to ^ i) & ~31 ? nxt.page : cur.page, to, st);
            if (++st == NST) st = 0, ph ^= 1;
        }

        // the warps' parts: (m, l) and o in units of 2^m, through the ring's space
        constexpr int OS = HD + 4;  // floats of a row there (rows 2 t of a warp's stores in distinct banks)
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                float y = l[n][e];
#pragma unroll
                for (int k = 4; k < 32; k *= 2) y += __shfl_xor_sync(0xffffffffu, y, k);
                if (g == 0) ml[warp][0][8 * n + 2 * t + e] = m[n][e], ml[warp][1][8 * n + 2 * t + e] = y;
            }
        __syncthreads();
        float* os = reinterpret_cast<float*>(smem);  // [warp][RT][OS]
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int j = 0; j < NJ; j++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    os[((size_t)warp * RT + 8 * n + 2 * t + (e & 1)) * OS + 16 * j + 8 * (e >> 1) + g] = o[n][j][e];
        __syncthreads();
        float* part = p.part + (size_t)(2 * blockIdx.x + (blockIdx.x == c0)) * RT * (HD + 2);
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
                const float4 y = *reinterpret_cast<const float4*>(os + ((size_t)w * RT + r) * OS + d);
                L = fmaf(ml[w][1][r], f, L);
                x.x = fmaf(y.x, f, x.x), x.y = fmaf(y.y, f, x.y), x.z = fmaf(y.z, f, x.z), x.w = fmaf(y.w, f, x.w);
            }
            if (ns == 1) {
                const float inv = L == 0.f ? 0.f : 1.0f / L;
                const int row = row0 + r;
                store4(a.out.at((size_t)sq.r0 + token(row), h * a.G + row - token(row) * a.G) + d, a.vec,
                       make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv));
            } else {
                float* y = part + (size_t)r * (HD + 2);
                *reinterpret_cast<float2*>(y + 2 + d) = make_float2(x.x, x.y);
                *reinterpret_cast<float2*>(y + 4 + d) = make_float2(x.z, x.w);
                if (d == 0) *reinterpret_cast<float2*>(y) = make_float2(M, L);
            }
        }
        bool last = false;
        if (ns > 1) {  // the CTA that comes last joins all parts, in their order
            __threadfence();
            __syncthreads();
            if (tid == 0) {
                last_cta = atomicAdd(p.tickets + c0, 1u) == ns - 1;
                if (last_cta) p.tickets[c0] = 0;
            }
            __syncthreads();
            last = last_cta;
        }
        if (last) {
            __threadfence();
            for (int i = tid; i < valid * (HD / 4); i += 32 * kStepWarps) {
                const int r = i / (HD / 4), d = 4 * (i % (HD / 4));
                float M = -INFINITY, L = 0.f;
                float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
                for (uint32_t k = 0; k < ns; k++) {
                    const float* y = p.part + ((size_t)(2 * (c0 + k) + (k == 0)) * RT + r) * (HD + 2);
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
                store4(a.out.at((size_t)sq.r0 + token(row), h * a.G + row - token(row) * a.G) + d, a.vec,
                       make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv));
            }
        }
        fence_proxy_async_smem();  // the ring's space goes back to the copies
        __syncthreads();
    }
}

template <int HD, typename T>
cudaError_t launch_kv8_step(const Kv8Attn<T>& a, const Kv8StepPlan& p, cudaStream_t st) {
    constexpr int smem = kStepWarps * StepRing<HD>::kStages * StepRing<HD>::kPairBytes;
    static_assert(smem >= kStepWarps * 16 * (HD + 4) * 4, "the ring holds the warps' parts");
    auto go = [&](auto* kernel, std::atomic<uint32_t>& done) {
        const cudaError_t e = kv8_smem_once(kernel, smem, p.device, done);
        if (e != cudaSuccess) return e;
        return launch_pdl(kernel, dim3(p.grid), dim3(32 * kStepWarps), smem, st, a, p);
    };
    static std::atomic<uint32_t> done1{0}, done2{0};
    return p.tiles == 1 ? go(&kv8_attn_step_kernel<HD, T, 1>, done1) : go(&kv8_attn_step_kernel<HD, T, 2>, done2);
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
