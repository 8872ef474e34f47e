// kv8.cu -- the 8-bit paged KV cache next to the decode path: norms and rotation of q and k rows,
// appending k and v rows to int8 pages, reading rows back, and the entry points of include/pox_cuda.h
// (the attention's kernels are in kv8_attn.cu).
#include <algorithm>
#include <exception>

#include "../../include/pox_cuda.h"
#include "api_internal.h"
#include "kv8.cuh"
#include "kv8_attn.h"
#include "kv8_math.cuh"

namespace pox {

// ---- norms of q and k with the rotation ----------------------------------------------------------
template <typename T>
struct QkArgs {
    RowsView<T> in[2], out[2];
    const __half* w[2];
    int heads[2];
    uint32_t rows;
    int hd;
    float eps;
    RopeView rope;
    const uint32_t* pos;
    int* err;
};

// Any shape: one warp per (row, head), a pass for the sum of squares and one for the pairs.
template <typename T>
__global__ void __launch_bounds__(256) qk_norm_rope_any_kernel(QkArgs<T> a) {
    pdl_wait();
    pdl_launch_dependents();
    const int nh = a.heads[0] + a.heads[1], lane = threadIdx.x & 31;
    const unsigned long long item = (unsigned long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (item >= (unsigned long long)a.rows * nh) return;
    const uint32_t r = (uint32_t)(item / nh);
    int h = (int)(item % nh);
    const int side = h >= a.heads[0];
    if (side) h -= a.heads[0];
    const int rot = a.rope.rot, half = rot / 2;
    const uint32_t p = rot ? a.pos[r] : 0;
    if (rot && p >= a.rope.positions) {
        if (lane == 0) atomicOr(a.err, kErrRopePos);
        return;
    }
    const T* x = a.in[side].at(r, h);
    T* y = a.out[side].at(r, h);
    const __half* w = a.w[side];
    float inv = 1.f;
    if (w) {
        float ss = 0.f;
        for (int d = lane; d < a.hd; d += 32) {
            const float v = to_f32(x[d]);
            ss = fmaf(v, v, ss);
        }
        inv = 1.0f / sqrtf(warp_sum(ss) / (float)a.hd + a.eps);
    }
    auto val = [&](int d) { return w ? to_f32(x[d]) * inv * __half2float(w[d]) : to_f32(x[d]); };
    for (int i = lane; i < half; i += 32) {
        const int d0 = a.rope.half ? i : 2 * i, d1 = a.rope.half ? i + half : 2 * i + 1;
        const float2 v = rope_turn(val(d0), val(d1), a.rope.table[(size_t)p * half + i]);
        y[d0] = from_f32<T>(v.x);
        y[d1] = from_f32<T>(v.y);
    }
    for (int d = rot + lane; d < a.hd; d += 32) y[d] = from_f32<T>(val(d));
}

// Bound by HBM (each element once in, once out): 16384 rows of 64 + 8 heads of 128, bf16, in 111 us, 84 % of the measured
// copy rate. A few rows are bound by the launch: 4 us on the device up to some hundred rows.
// 16 bytes a load: of the L = hd / (2 V) lanes of a head (V elements in 16 bytes), lane c holds the V dims from c V and
// the V dims from rot / 2 + c V, so that both kinds of pairs lie within a lane, and what is not rotated in order behind.
// A warp takes 32 / L heads of a row at once and `steps` such groups of it and keeps the row's cosines and sines and the
// norm's weights meanwhile. kQkAhead groups are on their way to shared memory, each lane's pieces to a place of its own
// (held in registers, two of them left too few bytes in flight for HBM). All arithmetic goes two elements to an
// instruction: at one each, the issue slots were as busy as the memory.
constexpr int kQkAhead = 4;
template <typename T, int L, bool HALF>
__global__ void __launch_bounds__(256, 3) qk_norm_rope_kernel(QkArgs<T> a, int steps, int groups) {
    constexpr int V = 16 / sizeof(T), HW = 32 / L, P = V / 2;
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31, c = lane % L, nh = a.heads[0] + a.heads[1], rot = a.rope.rot;
    const unsigned long long item = (unsigned long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    const uint32_t r = (uint32_t)div_u64(item, groups);
    if (r >= a.rows) return;
    const int h0 = (int)(item - (unsigned long long)r * groups) * steps * HW + lane / L, turn = c < rot / (2 * V);
    const int d0 = turn ? c * V : 2 * c * V, d1 = turn ? rot / 2 + c * V : d0 + V;
    const T* src[2] = {a.in[0].at(r, 0), a.in[1].at(r, 0)};
    __shared__ uint4 ahead[kQkAhead][2][256];
    auto fetch = [&](int k) {
        const int h = h0 + k * HW, side = h >= a.heads[0];
        if (k < steps && h < nh) {
            const T* p = (side ? src[1] : src[0]) + (size_t)(h - (side ? a.heads[0] : 0)) * a.in[side].head;
            cp16(smem_u32(&ahead[k % kQkAhead][0][threadIdx.x]), p + d0);
            cp16(smem_u32(&ahead[k % kQkAhead][1][threadIdx.x]), p + d1);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int k = 0; k < kQkAhead; k++) fetch(k);
    const uint32_t p = rot ? a.pos[r] : 0;
    if (rot && p >= a.rope.positions) {
        if (lane == 0) atomicOr(a.err, kErrRopePos);
        asm volatile("cp.async.wait_all;" ::: "memory");  // the copies on their way end before the CTA does
        return;
    }
    // HALF: cosines and sines of the V pairs, two to a register pair. Else (cos, sin) and (-sin, cos) of each of them:
    // the pairs of the lower piece, then of the upper one.
    uint64_t cs[V], sn[HALF ? 1 : V];
    if (turn) {
        const float2* t = a.rope.table + (size_t)p * (rot / 2);
        if constexpr (HALF) {
#pragma unroll
            for (int i = 0; i < P; i++) {
                const float4 q = __ldg(reinterpret_cast<const float4*>(t + c * V) + i);
                cs[i] = pair2(q.x, q.z);
                cs[P + i] = pair2(q.y, q.w);
            }
        } else {
#pragma unroll
            for (int i = 0; i < V; i++) {
                const float2 q = __ldg(t + (i < P ? c * P + i : (rot / 2 + c * V) / 2 + i - P));
                cs[i] = pair2(q.x, q.y);
                sn[i] = pair2(-q.y, q.x);
            }
        }
    }
    uint64_t w[2][P];
    int wside = -1;
    auto finish = [&](int k) {
        const int h = h0 + k * HW, side = h >= a.heads[0];
        const bool live = h < nh;
        asm volatile("cp.async.wait_group %0;" ::"n"(kQkAhead - 1) : "memory");
        uint64_t v[2][P], ss = 0;
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const uint4 x = live ? ahead[k % kQkAhead][u][threadIdx.x] : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int e = 0; e < P; e++) {
                v[u][e] = pair2(elem16<T>(x, 2 * e), elem16<T>(x, 2 * e + 1));
                ss = fma2(v[u][e], v[u][e], ss);
            }
        }
        float sum = both(ss).x + both(ss).y;
#pragma unroll
        for (int o = L / 2; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (!live) return;
        if (a.w[side]) {
            if (side != wside) {
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const uint32_t* q = reinterpret_cast<const uint32_t*>(a.w[side] + (u ? d1 : d0));
#pragma unroll
                    for (int e = 0; e < P; e++) {
                        const uint32_t g = __ldg(q + e);
                        const float2 f = unpack_f16(g);
                        w[u][e] = pair2(f.x, f.y);
                    }
                }
                wside = side;
            }
            // 1 / sqrt by the approximation and one step of Newton's method
            const float y = sum / (float)a.hd + a.eps, z = rsqrtf(y);
            const float inv = y > 0x1p-120f && y < INFINITY ? fmaf(0.5f * z, fmaf(-y * z, z, 1.0f), z) : 1.0f / sqrtf(y);
            const uint64_t f = pair2(inv, inv);
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int e = 0; e < P; e++) v[u][e] = mul2(mul2(v[u][e], f), w[u][e]);
        }
        if (turn) {
#pragma unroll
            for (int e = 0; e < P; e++) {
                if constexpr (HALF) {
                    const uint64_t lo = v[0][e], hi = v[1][e], z = mul2(hi, cs[P + e]);
                    v[0][e] = fma2(lo, cs[e], z ^ 0x8000000080000000ull);
                    v[1][e] = fma2(lo, cs[P + e], mul2(hi, cs[e]));
                } else {
#pragma unroll
                    for (int u = 0; u < 2; u++) {  // (a, b) -> a (cos, sin) + b (-sin, cos)
                        const float2 y = both(v[u][e]);
                        v[u][e] = fma2(pair2(y.x, y.x), cs[u * P + e], mul2(pair2(y.y, y.y), sn[u * P + e]));
                    }
                }
            }
        }
        T* y = a.out[side].at(r, h - (side ? a.heads[0] : 0));
#pragma unroll
        for (int u = 0; u < 2; u++) {
            uint32_t t[4];
#pragma unroll
            for (int e = 0; e < P; e++) {
                const float2 q = both(v[u][e]);
                if constexpr (sizeof(T) == 4) t[2 * e] = __float_as_uint(q.x), t[2 * e + 1] = __float_as_uint(q.y);
                else t[e] = pack2<T>(q.x, q.y);
            }
            *reinterpret_cast<uint4*>(y + (u ? d1 : d0)) = make_uint4(t[0], t[1], t[2], t[3]);
        }
    };
    for (int k = 0; k < steps; k++) {
        finish(k);
        fetch(k + kQkAhead);  // into the place just read
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
}

// ---- append ----------------------------------------------------------------------------------------
template <typename T>
struct AppendArgs {
    Kv8Cache c;
    Kv8Batch b;
    RowsView<const T> x[2];
    RopeView rope;
    int* err;
};

// What a unit of the append and read kernels works on: one page of one kv head, k or v.
struct PageUnit {
    SeqSpan sp;
    int page, first, last;  // its slots first .. last - 1 are rows of the batch
    size_t row;             // the row of slot `first`
    int blk;                // its block-table entry as found
    int8_t* bytes;          // the page of the kv head
    float* scale;
};
// The unit of page item `item` (the warp's), its entry loaded but not looked at; false (reported) if the batch is at
// fault. A sequence without a page of that number has first >= last.
__device__ __forceinline__ bool page_unit(const Kv8Batch& b, uint32_t item, PageUnit& o, int* err) {
    const uint32_t s = b.row_starts ? find_seq(b, item, [&](uint32_t q) { return page_base(b, q); }) : item;
    o.first = kPage, o.last = 0, o.page = 0, o.row = 0, o.blk = 0, o.bytes = nullptr;
    if (!seq_span(b, s, o.sp, err)) return false;
    const int begin = o.sp.ctx - o.sp.n, p0 = max(begin, 0);
    o.page = p0 / kPage + (int)(item - page_base(b, s));
    if (o.sp.ctx <= p0 || o.page * kPage >= o.sp.ctx) return true;
    o.first = max(p0 - o.page * kPage, 0), o.last = min(o.sp.ctx - o.page * kPage, kPage);
    o.row = (size_t)o.sp.r0 + (o.page * kPage + o.first - begin);
    o.blk = b.btab[(size_t)s * b.mbps + o.page];
    return true;
}
// Where the unit's page lies; false (reported) if the entry is out of range.
template <int HD>
__device__ __forceinline__ bool page_resolve(const Kv8Cache& c, int h, int side, PageUnit& o, int* err) {
    if (o.first >= o.last) return false;
    if (o.blk < 0 || (uint32_t)o.blk >= c.num_blocks) {
        atomicOr(err, kErrAttnPage);
        return false;
    }
    const size_t p = (size_t)o.blk * c.kvh + h;
    o.bytes = c.pages + p * (2 * kPage * HD);
    o.scale = c.scales + p * 2 + side;
    return true;
}

// The larger of m and |x|, NaN if either is one.
__device__ __forceinline__ float max_abs(float m, float x) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(m), "f"(fabsf(x)));
    return r;
}

// rint(x / s) as a byte, two at once (low 8 bits of q0 and q1): the quotient by Markstein's method (y = x r with r the
// rounded reciprocal, then y + (x - y s) r), the rounding by adding 1.5 * 2^23, whose sum's low byte is the two's
// complement of the whole number. s2 = (-s, -s), r2 = (r, r).
__device__ __forceinline__ void quantise2(float x0, float x1, uint64_t s2, uint64_t r2, uint32_t& q0, uint32_t& q1) {
    const uint64_t x = pair2(x0, x1), y = mul2(x, r2);
    const uint64_t z = add2(fma2(fma2(y, s2, x), r2, y), pair2(12582912.0f, 12582912.0f));
    asm("mov.b64 {%0, %1}, %2;" : "=r"(q0), "=r"(q1) : "l"(z));
}
__device__ __forceinline__ uint32_t pack_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return prmt(prmt(a, b, 0x0040), prmt(c, d, 0x0040), 0x5410);
}

// How the append reads rows and turns k. kAny goes element by element and finds partners in memory; the others load
// four elements at once and turn pairs within a lane (interleaved) or between lanes (halves of whole lanes).
enum { kTurnAny = 0, kTurnNone = 1, kTurnHalf = 2, kTurnPairs = 3 };

// Rows in once, bytes out once: a 16381-token f32 prompt (8 kv heads of 128, 176 MB with the rotation's table) in 44 us,
// 61 % of the measured copy rate: the chain of a unit (its rows, their turn, the maximum, the bytes) with 5 CTAs to an SM
// to cover it, and the arithmetic beside it. A decode step (5 us on the device) and a ragged batch of 8000 rows (9.6)
// are that chain once or a few times.
// A unit (page, kv head, side) is taken by two groups of HD / 4 lanes, lane c of group `hi` on dims 4 c .. 4 c + 3 of
// tokens 8 hi .. 8 hi + 7, whose rows are all in flight at once (with all 16 tokens on a lane, 168 registers left 12
// warps to an SM: no faster; a loop over the heads that fetches ahead: 66 us). The page's new rows set the scale, its
// older slots follow if the scale grew. A lane's four dims make a word of each K row and 8 bytes of each of four V rows.
template <int HD, typename T, int TURN>
__global__ void __launch_bounds__(128, 5) kv8_append_kernel(AppendArgs<T> a, uint32_t ctas) {
    constexpr int L = HD / 4, UC = 128 / (2 * L), NT = kPage / 2;
    pdl_wait();
    pdl_launch_dependents();
    if (check_batch(a.b, a.err)) return;
    __shared__ float red[4];
    const int lane = threadIdx.x & 31, c = threadIdx.x % L, hi = threadIdx.x / L & 1, t0 = NT * hi;
    const uint32_t item = blockIdx.x / ctas;
    const int u = (blockIdx.x - item * ctas) * UC + threadIdx.x / (2 * L), side = u >= a.c.kvh,
              h = min(u - side * a.c.kvh, a.c.kvh - 1);
    PageUnit o;
    bool live = page_unit(a.b, item, o, a.err) && u < 2 * a.c.kvh && o.first < o.last;
    const int rot = TURN == kTurnNone || side ? 0 : a.rope.rot, half = rot / 2, pos0 = o.page * kPage + t0;
    // a page with a row outside the table stays as it is, v too
    if (live && TURN != kTurnNone && a.rope.rot && (uint32_t)(o.page * kPage + o.last - 1) >= a.rope.positions) {
        if (c == 0) atomicOr(a.err, kErrRopePos);
        live = false;
    }
    const int first = live ? o.first - t0 : 0, last = live ? o.last - t0 : 0;  // in this lane's tokens
    auto in = [&](int t) { return t >= first && t < last; };
    const size_t ld = a.x[side].row;
    const T* x = a.x[side].at(live ? o.row : 0, h) - (ptrdiff_t)first * (ptrdiff_t)ld;  // of token t0, if it is a row
    Raw4<T> raw[NT];
#pragma unroll
    for (int t = 0; t < NT; t++)
        if (in(t)) raw[t].template load<TURN != kTurnAny>(x + t * (ptrdiff_t)ld + 4 * c);
    live = live && page_resolve<HD>(a.c, h, side, o, a.err);
    const bool whole = o.first == 0 && o.last == kPage;
    const float old = live && o.first ? *o.scale : 0.f;
    uint2 ov[4];  // older bytes of V (this lane's dims and tokens), where the page is not written whole
    if (live && side && !whole)
#pragma unroll
        for (int e = 0; e < 4; e++) ov[e] = *reinterpret_cast<const uint2*>(o.bytes + kv8_v_off<HD>(t0, 4 * c + e));
    float v[NT][4];
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
        for (int e = 0; e < 4; e++) v[t][e] = in(t) ? to_f32(raw[t].v[e]) : 0.f;
    if constexpr (TURN == kTurnHalf || TURN == kTurnPairs) {
        const bool mine = 4 * c < rot, low = 4 * c < half;
        const int from = !mine ? lane : low ? lane + rot / 8 : lane - rot / 8;
#pragma unroll
        for (int tc = 0; tc < NT; tc += 4) {  // (cos, sin) of four rows in flight
            if (!__any_sync(0xffffffffu, rot && last > tc && first < tc + 4)) continue;
            float4 cs[4][2];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int t = tc + i;
                if (mine && in(t)) {
                    const int at = TURN == kTurnHalf ? 4 * c - (low ? 0 : half) : 2 * c;
                    const float4* q = reinterpret_cast<const float4*>(a.rope.table + (size_t)(pos0 + t) * half + at);
                    cs[i][0] = __ldg(q);
                    if (TURN == kTurnHalf) cs[i][1] = __ldg(q + 1);
                }
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int t = tc + i;
                const float2* q = reinterpret_cast<const float2*>(cs[i]);
                if (TURN == kTurnHalf) {
                    float w[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) w[e] = __shfl_sync(0xffffffffu, v[t][e], from);
                    if (mine && in(t))
#pragma unroll
                        for (int e = 0; e < 4; e++)  // rope_turn's half that this lane keeps
                            v[t][e] = __fadd_rn(__fmul_rn(v[t][e], q[e].x), __fmul_rn(w[e], low ? -q[e].y : q[e].y));
                } else if (mine && in(t)) {
#pragma unroll
                    for (int e = 0; e < 4; e += 2) {
                        const float2 y = rope_turn(v[t][e], v[t][e + 1], q[e / 2]);
                        v[t][e] = y.x, v[t][e + 1] = y.y;
                    }
                }
            }
        }
    } else if (TURN == kTurnAny && rot) {
#pragma unroll
        for (int t = 0; t < NT; t++) {
            if (!in(t)) continue;
            const T* xr = x + t * (ptrdiff_t)ld;
            const float2* tab = a.rope.table + (size_t)(pos0 + t) * half;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int d = 4 * c + e;
                if (d >= rot) continue;
                const bool lo = a.rope.half ? d < half : !(d & 1);
                const int p = a.rope.half ? (lo ? d + half : d - half) : d ^ 1;
                const float2 cs = tab[a.rope.half ? (lo ? d : p) : d / 2];
                const float own = to_f32(xr[d]), other = to_f32(xr[p]);
                v[t][e] = lo ? rope_turn(own, other, cs).x : rope_turn(other, own, cs).y;
            }
        }
    }
    // the unit's largest magnitude: over the lanes of both groups
    auto joined = [&](float m) {
#pragma unroll
        for (int k = (L == 32 ? 16 : L); k; k >>= 1) m = max_abs(m, __shfl_xor_sync(0xffffffffu, m, k));
        if constexpr (L == 32) {
            if (lane == 0) red[threadIdx.x >> 5] = m;
            __syncthreads();
            m = max_abs(m, red[threadIdx.x >> 5 ^ 1]);
        }
        return m;
    };
    float m = 0.f;
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
        for (int e = 0; e < 4; e++) m = max_abs(m, v[t][e]);
    m = joined(m);
    // rare: infinities saturate, NaN is 0, neither sets the scale; and scales whose reciprocal would leave the range
    float up = 1.f;
    if (__syncthreads_or(!(m < 0x1p120f) || (m > 0.f && m < 0x1p-90f) || (old > 0.f && old < 0x1p-100f))) {
        m = 0.f;
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (fabsf(v[t][e]) < INFINITY) m = fmaxf(m, fabsf(v[t][e]));
        m = joined(m);
        const float now = fmaxf(old, __fdiv_rn(m, 127.f));
        up = now < 0x1p-64f ? 0x1p64f : now > 0x1p64f ? 0x1p-64f : 1.f;
        const float most = 127.f * (now * up);  // (a subnormal scale is coarse: up to 190 such steps in an element)
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float y = v[t][e];
                v[t][e] = y != y ? 0.f : fminf(fmaxf(y * up, -most), most);
            }
    }
    if (!live) return;
    const float now = fmaxf(old, __fdiv_rn(m, 127.f));
    const bool grew = o.first && now > old;
    const float ratio = grew ? __fdiv_rn(old, now) : 1.f;
    const float s = now > 0.f ? now * up : 1.f, rs = __frcp_rn(s);
    const uint64_t s2 = pair2(-s, -s), r2 = pair2(rs, rs);
    auto older = [&](uint32_t w, int n) {  // the first n bytes of a word to the new scale
        uint32_t q[4];
#pragma unroll
        for (int e = 0; e < 4; e++)
            q[e] = e < n ? __float_as_uint(__fadd_rn(__fmul_rn((float)(int8_t)(w >> 8 * e), ratio), 12582912.0f))
                         : w >> 8 * e;
        return pack_bytes(q[0], q[1], q[2], q[3]);
    };
    if (side == 0) {
        if (grew)
            for (int t = 0; t < min(first, NT); t++) {
                uint32_t* w = reinterpret_cast<uint32_t*>(o.bytes + kv8_k_off<HD>(t0 + t, 4 * c));
                *w = older(*w, 4);
            }
#pragma unroll
        for (int t = 0; t < NT; t++)
            if (in(t)) {
                uint32_t q[4];
                quantise2(v[t][0], v[t][1], s2, r2, q[0], q[1]);
                quantise2(v[t][2], v[t][3], s2, r2, q[2], q[3]);
                *reinterpret_cast<uint32_t*>(o.bytes + kv8_k_off<HD>(t0 + t, 4 * c)) =
                    pack_bytes(q[0], q[1], q[2], q[3]);
            }
    } else if (whole || grew || (first < NT && last > 0)) {
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
            uint32_t w[2][2];
#pragma unroll
            for (int k = 0; k < 2; k++) {
                uint32_t q[2][4];
#pragma unroll
                for (int t = 0; t < 4; t++) quantise2(v[4 * k + t][e], v[4 * k + t][e + 1], s2, r2, q[0][t], q[1][t]);
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    w[i][k] = pack_bytes(q[i][0], q[i][1], q[i][2], q[i][3]);
                    if (!whole) {
                        const uint32_t b = k ? ov[e + i].y : ov[e + i].x, keep = grew ? older(b, first - 4 * k) : b;
                        uint32_t mask = 0;  // bytes of slots first .. last - 1
#pragma unroll
                        for (int t = 0; t < 4; t++) mask |= in(4 * k + t) ? 0xffu << 8 * t : 0u;
                        w[i][k] = (w[i][k] & mask) | (keep & ~mask);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < 2; i++)
                *reinterpret_cast<uint2*>(o.bytes + kv8_v_off<HD>(t0, 4 * c + e + i)) = make_uint2(w[i][0], w[i][1]);
        }
    }
    if (c == 0 && hi == 0) *o.scale = now;
}

// ---- reading rows back -------------------------------------------------------------------------------
// The append's units the other way round, one group of HD / 4 lanes to all tokens of a unit. The unit of a sequence's
// first page also clears its padding rows. Bound by HBM: a 16381-token prompt (8 kv heads of
// 128) to f32 rows, 168 MB, in 29 us, 88 % of the measured copy rate; a decode step by the launch, 5 us on the device.
template <int HD, typename T>
__global__ void __launch_bounds__(128) kv8_read_kernel(Kv8Cache cache, Kv8Batch b, RowsView<T> k, RowsView<T> v,
                                                       uint32_t ctas, int vec, int* err) {
    constexpr int L = HD / 4;
    pdl_wait();
    pdl_launch_dependents();
    if (check_batch(b, err)) return;
    const uint32_t item = blockIdx.x / ctas;
    const int c = threadIdx.x % L, u = (blockIdx.x - item * ctas) * (128 / L) + threadIdx.x / L, side = u >= cache.kvh,
              h = u - side * cache.kvh;
    PageUnit o;
    if (!page_unit(b, item, o, err) || u >= 2 * cache.kvh) return;
    const RowsView<T>& out = side ? v : k;
    const int begin = o.sp.ctx - o.sp.n;
    if (begin < 0 && o.page == 0)
        for (int i = 0; i < min(-begin, o.sp.n); i++)
            store4(out.at((size_t)o.sp.r0 + i, h) + 4 * c, vec, make_float4(0.f, 0.f, 0.f, 0.f));
    if (!page_resolve<HD>(cache, h, side, o, err)) return;
    const float s = *o.scale;
    uint32_t w[kPage];  // K: the four dims of each token; V: four words of each dim
    if (side == 0) {
#pragma unroll
        for (int t = 0; t < kPage; t++)
            if (t >= o.first && t < o.last) w[t] = *reinterpret_cast<const uint32_t*>(o.bytes + kv8_k_off<HD>(t, 4 * c));
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const uint4 x = *reinterpret_cast<const uint4*>(o.bytes + kv8_v_off<HD>(0, 4 * c + e));
            w[4 * e] = x.x, w[4 * e + 1] = x.y, w[4 * e + 2] = x.z, w[4 * e + 3] = x.w;
        }
    }
    T* y = out.at(o.row, h) + 4 * c;
#pragma unroll
    for (int t = 0; t < kPage; t++)
        if (t >= o.first && t < o.last) {
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                // 2^23 + (byte + 128), exactly
                const uint32_t q = side ? prmt(w[4 * e + t / 4], 0x4b000000u, 0x7440 + t % 4)
                                        : prmt(w[t], 0x4b000000u, 0x7440 + e);
                x[e] = __fmul_rn(__uint_as_float(q ^ 0x80u) - 8388736.0f, s);
            }
            store4(y + (size_t)(t - o.first) * out.row, vec, make_float4(x[0], x[1], x[2], x[3]));
        }
}

// ---- checks of arguments ------------------------------------------------------------------------------
static int esize(int dtype) { return dtype == POX_F32 ? 4 : dtype == POX_F16 || dtype == POX_BF16 ? 2 : 0; }

static int check_rows(const pox_rows* r, const char* what, uint32_t rows, uint32_t heads, uint32_t hd, bool written) {
    if (!r || !r->data) return set_error(POX_ERR_INVALID, "%s is NULL", what);
    const int es = esize(r->dtype);
    if (!es) return set_error(POX_ERR_UNSUPPORTED, "%s: dtype %d (supported: f32, f16, bf16)", what, r->dtype);
    if ((uintptr_t)r->data % es) return set_error(POX_ERR_INVALID, "%s is not aligned to its element", what);
    // the farthest element's offset has to fit the address space with room to spare
    const unsigned __int128 far = (unsigned __int128)(rows ? rows - 1 : 0) * r->row_stride +
                                  (unsigned __int128)(heads ? heads - 1 : 0) * r->head_stride + hd;
    if (far >= ((unsigned __int128)1 << 46))
        return set_error(POX_ERR_INVALID, "%s: strides out of range", what);
    if (written) {
        const bool apart =
            ((heads <= 1 || r->head_stride >= hd) &&
             (rows <= 1 || r->row_stride >= (uint64_t)(heads - 1) * r->head_stride + hd)) ||
            ((rows <= 1 || r->row_stride >= hd) &&
             (heads <= 1 || r->head_stride >= (uint64_t)(rows - 1) * r->row_stride + hd));
        if (!apart) return set_error(POX_ERR_INVALID, "%s: rows or heads of an output overlap", what);
    }
    return POX_OK;
}

static int check_rope(const pox_rope* r, uint32_t hd) {
    if (!r || !r->rot_dim) return POX_OK;
    if (r->rot_dim % 2 || r->rot_dim > hd)
        return set_error(POX_ERR_INVALID, "rot_dim %u is not an even number up to the head's %u", r->rot_dim, hd);
    if (!r->table || !r->positions) return set_error(POX_ERR_INVALID, "rotation table is NULL or empty");
    if ((uintptr_t)r->table % 8) return set_error(POX_ERR_INVALID, "rotation table is not 8-byte aligned");
    if (r->style != POX_ROPE_INTERLEAVED && r->style != POX_ROPE_HALF)
        return set_error(POX_ERR_UNSUPPORTED, "rotation style %d", r->style);
    return POX_OK;
}

static RopeView rope_view(const pox_rope* r) {
    RopeView v{nullptr, 0, 0, 0};
    if (r && r->rot_dim)
        v = RopeView{reinterpret_cast<const float2*>(r->table), r->positions, (int)r->rot_dim,
                     r->style == POX_ROPE_HALF};
    return v;
}

template <typename T>
static RowsView<T> rows_view(const pox_rows& r) {
    return RowsView<T>{static_cast<T*>(r.data), (size_t)r.row_stride, (size_t)r.head_stride};
}

static int check_cache(const pox_kv8_cache* c, const pox_kv8_batch* b) {
    if (!c || !b) return set_error(POX_ERR_INVALID, "cache or batch is NULL");
    if (b->rows == 0 || b->seqs == 0) return POX_OK;
    if (!c->pages || !c->scales || !b->ctx_lens || !b->block_tables)
        return set_error(POX_ERR_INVALID, "NULL device pointer in cache or batch");
    if (!c->num_blocks || !c->kv_heads || !b->max_blocks_per_seq || !b->max_rows)
        return set_error(POX_ERR_INVALID, "zero num_blocks, kv_heads, max_blocks_per_seq or max_rows");
    if (c->head_dim != 32 && c->head_dim != 64 && c->head_dim != 128)
        return set_error(POX_ERR_UNSUPPORTED, "head_dim %u (supported: 32, 64, 128)", c->head_dim);
    if (((uintptr_t)c->pages & 15) || ((uintptr_t)c->scales & 7))
        return set_error(POX_ERR_INVALID, "pages must be 16-byte, scales 8-byte aligned");
    if (((uintptr_t)b->ctx_lens | (uintptr_t)b->block_tables | (uintptr_t)b->row_starts) & 3)
        return set_error(POX_ERR_INVALID, "batch arrays must be 4-byte aligned");
    if (!b->row_starts && b->rows != b->seqs)
        return set_error(POX_ERR_INVALID, "%u rows for %u sequences of one row", b->rows, b->seqs);
    if (b->max_blocks_per_seq > (1u << 26) || b->max_ctx > b->max_blocks_per_seq * (uint64_t)kPage)
        return set_error(POX_ERR_INVALID, "max_ctx %u is beyond %u pages", b->max_ctx, b->max_blocks_per_seq);
    if (c->kv_heads > 4096 || b->rows > (1u << 26) || b->seqs > (1u << 22))
        return set_error(POX_ERR_UNSUPPORTED, "%u kv heads / %u rows / %u sequences", c->kv_heads, b->rows, b->seqs);
    return POX_OK;
}

static Kv8Cache cache_view(const pox_kv8_cache* c) {
    return Kv8Cache{c->pages, c->scales, c->num_blocks, (int)c->kv_heads};
}
static Kv8Batch batch_view(const pox_kv8_batch* b) {
    // as many rows as sequences and at most one each: one each, and no search on the device
    const bool single = b->max_rows == 1 && b->rows == b->seqs;
    return Kv8Batch{single ? nullptr : b->row_starts, b->ctx_lens, b->block_tables,       b->seqs, b->rows,
                    std::min(b->max_rows, b->rows),   b->max_ctx,  b->max_blocks_per_seq,
                    single ? b->row_starts : nullptr};
}

constexpr int kPromptRows = 64;

// Which of the attention's kernels a batch of more rows should take, from the bounds that the host knows. The step
// kernel spreads rows by 16 and the context over the whole GPU, a page of a tile at about 0.65 ns (head dim 128; 64:
// 0.46); a CTA of the prompt kernel walks the context for 256 rows, 128 tokens in 2.75 us (up to 128 rows 2.35; head dim
// 64: 2.35 and 2.05). Both ways measured, bf16, 8 kv heads of 128 with 4 query heads each, step against prompt kernel:
// one sequence of 128 rows at 4096 tokens 61 us against 87, of 512 at 512 43 against 30; eight of 32 rows at 4096 108
// against 77, of 16 61 against 63; one of 256 at 32768 626 against 544.
static bool prompt_is_faster(const pox_kv8_cache* c, const pox_kv8_batch* b, int G, int sms) {
    const double rows = (double)b->rows * G, most = (double)std::min(b->max_rows, b->rows) * G;
    const bool wide = c->head_dim == 128;
    const double step = c->kv_heads * (rows / 16 + b->seqs / 2.0) * (b->max_ctx / 16.0) * (wide ? 0.65 : 0.46);
    const double ctas = c->kv_heads * (rows / 256 + b->seqs / 2.0);
    const double tile = most <= 128 ? (wide ? 2350 : 2050) : (wide ? 2750 : 2350);
    return std::max(1.0, ctas / sms) * (b->max_ctx / 128.0) * tile < step;
}

// The stream's places for the parts of items that a plan cuts, and their tickets: made by its first call, as large as any
// plan on this device asks for, and not moved (a captured graph holds their addresses). Those of a stream that is
// known to be destroyed go to the next new one, after a pox_cuda_synchronize and unless they were captured. A call that
// does not use them (`used` false) makes them all the same, so that any first call readies the stream for a capture.
static int kv8_scratch(pox_cuda_ctx* ctx, cudaStream_t st, Kv8StepPlan& p, bool used) {
    try {
        std::lock_guard<std::mutex> lk(ctx->mu);
        auto same_handle = [&](const Kv8Scratch& x) {
            return x.handle == st && (st != cudaStreamPerThread || x.thread == std::this_thread::get_id()) && !x.over;
        };
        cudaStreamCaptureStatus cs = cudaStreamCaptureStatusNone;
        cudaError_t e = cudaStreamIsCapturing(st, &cs);
        if (e != cudaSuccess) return cuda_error(e, "stream of kv8_attention");
        if (cs != cudaStreamCaptureStatusNone) {  // (a stream's id is not to be had while it is captured)
            if (!used) return POX_OK;
            for (auto& k : ctx->kv8)
                if (same_handle(k.second) && k.second.tickets) {
                    k.second.captured = true;
                    p.part = k.second.part, p.tickets = k.second.tickets;
                    return POX_OK;
                }
            return set_error(POX_ERR_INVALID, "the parts' places must be allocated by a call before stream capture");
        }
        unsigned long long id = 0;
        e = cudaStreamGetId(st, &id);
        if (e != cudaSuccess) return cuda_error(e, "stream of kv8_attention");
        auto at = ctx->kv8.find(id);
        if (at == ctx->kv8.end() || !at->second.tickets) {
            if (at == ctx->kv8.end()) {
                auto idle = ctx->kv8.end();
                for (auto k = ctx->kv8.begin(); k != ctx->kv8.end(); ++k) {
                    if (same_handle(k->second)) k->second.over = true, k->second.over_since = ctx->syncs;
                    if (k->second.idle) idle = k;
                }
                if (idle == ctx->kv8.end()) {
                    at = ctx->kv8.emplace(id, Kv8Scratch()).first;
                } else {
                    float* part = idle->second.part;
                    auto node = ctx->kv8.extract(idle);
                    node.key() = id;
                    node.mapped() = Kv8Scratch();
                    node.mapped().part = part;
                    at = ctx->kv8.insert(std::move(node)).position;
                }
                at->second.handle = st;
                at->second.thread = std::this_thread::get_id();
            }
            Kv8Scratch& k = at->second;
            const size_t tickets = (size_t)Kv8StepPlan::most_ctas(ctx->num_sms) * sizeof(uint32_t);
            if (!k.part) {
                e = cudaMalloc(&k.part, Kv8StepPlan::most_part_bytes(ctx->num_sms) + tickets);
                if (e != cudaSuccess) return cuda_error(e, "split partials");
            }
            uint32_t* t = reinterpret_cast<uint32_t*>(reinterpret_cast<uint8_t*>(k.part) +
                                                      Kv8StepPlan::most_part_bytes(ctx->num_sms));
            e = cudaMemsetAsync(t, 0, tickets, st);
            if (e != cudaSuccess) return cuda_error(e, "split partials");
            k.tickets = t;
        }
        p.part = at->second.part;
        p.tickets = at->second.tickets;
    } catch (const std::exception& x) {  // (no exception crosses the C boundary)
        return set_error(POX_ERR_OOM, "split partials: %s", x.what());
    }
    return POX_OK;
}

template <typename T>
static cudaError_t launch_qk(pox_cuda_ctx* ctx, const pox_qk_norm_rope* a, cudaStream_t st) {
    QkArgs<T> k;
    k.in[0] = rows_view<T>(a->q), k.in[1] = rows_view<T>(a->k);
    k.out[0] = rows_view<T>(a->q_out), k.out[1] = rows_view<T>(a->k_out);
    k.w[0] = reinterpret_cast<const __half*>(a->q_norm), k.w[1] = reinterpret_cast<const __half*>(a->k_norm);
    k.heads[0] = (int)a->heads, k.heads[1] = (int)a->kv_heads;
    k.rows = a->rows, k.hd = (int)a->head_dim, k.eps = a->eps;
    k.rope = rope_view(&a->rope);
    k.pos = a->positions, k.err = ctx->err_dev;
    const int V = 16 / (int)sizeof(T), hd = (int)a->head_dim, L = hd / (2 * V), nh = (int)(a->heads + a->kv_heads);
    bool vec = hd % (2 * V) == 0 && k.rope.rot % (2 * V) == 0 && (L & (L - 1)) == 0 && L >= 2 && L <= 32 &&
               ((uintptr_t)k.rope.table & 15) == 0;
    for (int i = 0; i < 2; i++)
        if (k.heads[i])
            vec = vec && (((uintptr_t)k.in[i].data | (uintptr_t)k.out[i].data | (uintptr_t)k.w[i]) & 15) == 0 &&
                  ((k.in[i].row | k.in[i].head | k.out[i].row | k.out[i].head) % V) == 0;
    if (!vec) {
        const unsigned long long grid = ((unsigned long long)a->rows * nh + 7) / 8;
        if (grid > 0x7fffffffu) return cudaErrorInvalidConfiguration;
        return launch_pdl(qk_norm_rope_any_kernel<T>, dim3((unsigned)grid), dim3(256), 0, st, k);
    }
    // as many groups of heads to a warp as leave every SM its 32 warps
    const int all = (nh * L + 31) / 32;
    const int steps = (int)std::min<long long>(std::max<long long>((long long)a->rows * all / (32LL * ctx->num_sms), 1),
                                               std::min(all, 10));
    const int groups = (all + steps - 1) / steps;
    const unsigned long long grid = ((unsigned long long)a->rows * groups + 7) / 8;
    if (grid > 0x7fffffffu) return cudaErrorInvalidConfiguration;
    auto go = [&](auto* kernel) { return launch_pdl(kernel, dim3((unsigned)grid), dim3(256), 0, st, k, steps, groups); };
    auto by_lanes = [&](auto half) {
        constexpr bool H = decltype(half)::value;
        return L == 2 ? go(qk_norm_rope_kernel<T, 2, H>) : L == 4 ? go(qk_norm_rope_kernel<T, 4, H>)
             : L == 8 ? go(qk_norm_rope_kernel<T, 8, H>) : L == 16 ? go(qk_norm_rope_kernel<T, 16, H>)
                                                                    : go(qk_norm_rope_kernel<T, 32, H>);
    };
    return k.rope.half ? by_lanes(std::true_type()) : by_lanes(std::false_type());
}

static uint32_t page_items(const pox_kv8_batch* b) {
    return batch_view(b).row_starts ? (uint32_t)((b->rows + 30ull * b->seqs) / 16) : b->seqs;
}
// four elements of any (row, head) at once
static int vec4(const pox_rows* r) {
    return (uintptr_t)r->data % (4 * esize(r->dtype)) == 0 && (r->row_stride | r->head_stride) % 4 == 0;
}

template <int HD, typename T>
static cudaError_t launch_append(pox_cuda_ctx* ctx, const pox_kv8_cache* c, const pox_kv8_batch* b, const pox_rows* k,
                                 const pox_rows* v, const pox_rope* rope, cudaStream_t st) {
    AppendArgs<T> a{cache_view(c), batch_view(b), {rows_view<const T>(*k), rows_view<const T>(*v)}, rope_view(rope),
                    ctx->err_dev};
    constexpr unsigned kUnits = 128 / (HD / 2);  // of a CTA
    const unsigned ctas = (2 * c->kv_heads + kUnits - 1) / kUnits;  // of a page item
    const unsigned long long grid = (unsigned long long)page_items(b) * ctas + (a.b.row_starts ? 1 : 0);
    if (grid > 0x7fffffffu) return cudaErrorInvalidConfiguration;
    const RopeView& r = a.rope;
    const bool vec = vec4(k) && vec4(v) && ((uintptr_t)r.table & 15) == 0;
    auto go = [&](auto* kernel) { return launch_pdl(kernel, dim3((unsigned)grid), dim3(128), 0, st, a, ctas); };
    return vec && !r.rot                      ? go(kv8_append_kernel<HD, T, kTurnNone>)
           : vec && r.half && r.rot % 8 == 0  ? go(kv8_append_kernel<HD, T, kTurnHalf>)
           : vec && !r.half && r.rot % 4 == 0 ? go(kv8_append_kernel<HD, T, kTurnPairs>)
                                              : go(kv8_append_kernel<HD, T, kTurnAny>);
}

template <int HD, typename T>
static cudaError_t launch_read(pox_cuda_ctx* ctx, const pox_kv8_cache* c, const pox_kv8_batch* b, const pox_rows* k,
                               const pox_rows* v, cudaStream_t st) {
    constexpr unsigned kUnits = 128 / (HD / 4);  // of a CTA
    const unsigned ctas = (2 * c->kv_heads + kUnits - 1) / kUnits;
    const Kv8Batch view = batch_view(b);
    const unsigned long long grid = (unsigned long long)page_items(b) * ctas + (view.row_starts ? 1 : 0);
    if (grid > 0x7fffffffu) return cudaErrorInvalidConfiguration;
    return launch_pdl(kv8_read_kernel<HD, T>, dim3((unsigned)grid), dim3(128), 0, st, cache_view(c), view,
                      rows_view<T>(*k), rows_view<T>(*v), ctas, vec4(k) && vec4(v), ctx->err_dev);
}

// f.template operator()<HD, T>() for the head dim and the rows' type
template <typename F>
static cudaError_t by_type(int dtype, F&& f) {
    return dtype == POX_F32 ? f(float()) : dtype == POX_F16 ? f(__half()) : f(__nv_bfloat16());
}
template <typename F>
static cudaError_t by_shape(uint32_t hd, int dtype, F&& f) {
    return by_type(dtype, [&](auto t) {
        return hd == 32    ? f(std::integral_constant<int, 32>(), t)
               : hd == 64 ? f(std::integral_constant<int, 64>(), t)
                          : f(std::integral_constant<int, 128>(), t);
    });
}

}  // namespace pox

using namespace pox;

extern "C" int pox_cuda_qk_norm_rope(pox_cuda_ctx* ctx, const pox_qk_norm_rope* a, void* stream) {
    if (!ctx || !a) return set_error(POX_ERR_INVALID, "ctx or args is NULL");
    if (a->rows == 0 || a->heads + (uint64_t)a->kv_heads == 0) return POX_OK;
    if (a->head_dim == 0 || a->head_dim % 2 || a->head_dim > 512)
        return set_error(POX_ERR_UNSUPPORTED, "head_dim %u (supported: even, up to 512)", a->head_dim);
    if (a->heads > 4096 || a->kv_heads > 4096 || a->rows > (1u << 26))
        return set_error(POX_ERR_UNSUPPORTED, "%u / %u heads, %u rows", a->heads, a->kv_heads, a->rows);
    const struct {
        const pox_rows *in, *out;
        uint32_t heads;
        const char *name, *out_name;
    } side[2] = {{&a->q, &a->q_out, a->heads, "q", "q_out"}, {&a->k, &a->k_out, a->kv_heads, "k", "k_out"}};
    const int dtype = a->heads ? a->q.dtype : a->k.dtype;
    for (const auto& s : side) {
        if (!s.heads) continue;
        int rc = check_rows(s.in, s.name, a->rows, s.heads, a->head_dim, false);
        if (!rc) rc = check_rows(s.out, s.out_name, a->rows, s.heads, a->head_dim, true);
        if (rc) return rc;
        if (s.in->dtype != dtype || s.out->dtype != dtype)
            return set_error(POX_ERR_INVALID, "rows of different types (%s)", s.name);
        if (s.in->data == s.out->data &&
            (s.in->row_stride != s.out->row_stride || s.in->head_stride != s.out->head_stride))
            return set_error(POX_ERR_INVALID, "%s in place needs the same strides", s.name);
    }
    int rc = check_rope(&a->rope, a->head_dim);
    if (rc) return rc;
    if (a->rope.rot_dim && !a->positions) return set_error(POX_ERR_INVALID, "positions is NULL");
    if (((uintptr_t)a->positions & 3) || ((uintptr_t)a->q_norm & 1) || ((uintptr_t)a->k_norm & 1))
        return set_error(POX_ERR_INVALID, "positions or norm weights are not aligned to their elements");
    cudaError_t e = cudaSetDevice(ctx->device);
    if (e != cudaSuccess) return cuda_error(e, "cudaSetDevice");
    cudaStream_t st = stream ? (cudaStream_t)stream : ctx->stream;
    e = by_type(dtype, [&](auto t) { return launch_qk<decltype(t)>(ctx, a, st); });
    return e == cudaSuccess ? POX_OK : cuda_error(e, "qk_norm_rope launch");
}

static int check_kv_rows(const pox_kv8_cache* c, const pox_kv8_batch* b, const pox_rows* k, const pox_rows* v,
                         bool written) {
    int rc = check_rows(k, "k", b->rows, c->kv_heads, c->head_dim, written);
    if (!rc) rc = check_rows(v, "v", b->rows, c->kv_heads, c->head_dim, written);
    if (!rc && k->dtype != v->dtype) rc = set_error(POX_ERR_INVALID, "k and v rows of different types");
    return rc;
}

extern "C" int pox_cuda_kv8_append(pox_cuda_ctx* ctx, const pox_kv8_cache* c, const pox_kv8_batch* b, const pox_rows* k,
                                   const pox_rows* v, const pox_rope* rope, void* stream) {
    if (!ctx) return set_error(POX_ERR_INVALID, "ctx is NULL");
    int rc = check_cache(c, b);
    if (rc || b->rows == 0 || b->seqs == 0) return rc;
    rc = check_kv_rows(c, b, k, v, false);
    if (!rc) rc = check_rope(rope, c->head_dim);
    if (rc) return rc;
    cudaError_t e = cudaSetDevice(ctx->device);
    if (e != cudaSuccess) return cuda_error(e, "cudaSetDevice");
    cudaStream_t st = stream ? (cudaStream_t)stream : ctx->stream;
    e = by_shape(c->head_dim, k->dtype, [&](auto hd, auto t) {
        return launch_append<decltype(hd)::value, decltype(t)>(ctx, c, b, k, v, rope, st);
    });
    return e == cudaSuccess ? POX_OK : cuda_error(e, "kv8_append launch");
}

extern "C" int pox_cuda_kv8_read(pox_cuda_ctx* ctx, const pox_kv8_cache* c, const pox_kv8_batch* b, const pox_rows* k,
                                 const pox_rows* v, void* stream) {
    if (!ctx) return set_error(POX_ERR_INVALID, "ctx is NULL");
    int rc = check_cache(c, b);
    if (rc || b->rows == 0 || b->seqs == 0) return rc;
    rc = check_kv_rows(c, b, k, v, true);
    if (rc) return rc;
    cudaError_t e = cudaSetDevice(ctx->device);
    if (e != cudaSuccess) return cuda_error(e, "cudaSetDevice");
    cudaStream_t st = stream ? (cudaStream_t)stream : ctx->stream;
    e = by_shape(c->head_dim, k->dtype, [&](auto hd, auto t) {
        return launch_read<decltype(hd)::value, decltype(t)>(ctx, c, b, k, v, st);
    });
    return e == cudaSuccess ? POX_OK : cuda_error(e, "kv8_read launch");
}

extern "C" int pox_cuda_kv8_attention(pox_cuda_ctx* ctx, const pox_kv8_cache* c, const pox_kv8_batch* b,
                                      const pox_rows* q, const pox_rows* out, uint32_t heads, float scale,
                                      void* stream) {
    if (!ctx) return set_error(POX_ERR_INVALID, "ctx is NULL");
    int rc = check_cache(c, b);
    if (rc || b->rows == 0 || b->seqs == 0) return rc;
    if (!heads || heads % c->kv_heads)
        return set_error(POX_ERR_INVALID, "%u heads over %u kv heads", heads, c->kv_heads);
    if (heads / c->kv_heads > 128)
        return set_error(POX_ERR_UNSUPPORTED, "%u query heads per kv head (at most 128)", heads / c->kv_heads);
    rc = check_rows(q, "q", b->rows, heads, c->head_dim, false);
    if (!rc) rc = check_rows(out, "out", b->rows, heads, c->head_dim, true);
    if (rc) return rc;
    if (q->dtype != out->dtype) return set_error(POX_ERR_INVALID, "q and out rows of different types");
    if (!(scale >= 0.f && scale < INFINITY)) return set_error(POX_ERR_INVALID, "scale %g", (double)scale);
    cudaError_t e = cudaSetDevice(ctx->device);
    if (e != cudaSuccess) return cuda_error(e, "cudaSetDevice");
    cudaStream_t st = stream ? (cudaStream_t)stream : ctx->stream;
    const int G = (int)(heads / c->kv_heads);
    const long long most = (long long)std::min(b->max_rows, b->rows) * G;
    if (most > 1 << 30)  // (the kernels count a sequence's rows in int)
        return set_error(POX_ERR_UNSUPPORTED, "%u rows of %d query heads", std::min(b->max_rows, b->rows), G);
    // Sequences of more rows than kPromptRows go to the tensor-memory kernel, where the whole batch is worth it; a batch
    // may hold both kinds, told apart on the device. All rows equal (or one sequence) means one kind.
    const bool prompt = c->head_dim != 32 && q->dtype != POX_F32 && most > kPromptRows &&
                        kv8_prompt_grid(batch_view(b), (int)c->kv_heads, G) <= 0x7fffffffu &&
                        prompt_is_faster(c, b, G, ctx->num_sms);
    const bool step = !prompt || (b->seqs > 1 && b->rows != (unsigned long long)b->seqs * b->max_rows);
    Kv8StepPlan plan = kv8_step_plan(batch_view(b), (int)c->kv_heads, (int)c->head_dim, G, ctx->num_sms,
                                     prompt ? kPromptRows : 0x7fffffff);
    plan.device = ctx->device;
    rc = kv8_scratch(ctx, st, plan, step);
    if (rc) return rc;
    const int vec = vec4(q) && vec4(out);
    e = by_shape(c->head_dim, q->dtype, [&](auto hd, auto t) {
        using T = decltype(t);
        const float s = (scale > 0.f ? scale : 1.0f / sqrtf((float)c->head_dim)) * 1.4426950408889634f;
        Kv8Attn<T> a{cache_view(c), batch_view(b), rows_view<const T>(*q), rows_view<T>(*out), G, s, vec, ctx->err_dev};
        constexpr int HD = decltype(hd)::value;
        cudaError_t r = cudaSuccess;
        if constexpr (HD != 32 && sizeof(T) == 2)
            if (prompt) r = launch_kv8_prompt<HD, T>(a, step ? kPromptRows + 1 : 1, ctx->device, st);
        if (r == cudaSuccess && step) r = launch_kv8_step<HD, T>(a, plan, st);
        return r;
    });
    return e == cudaSuccess ? POX_OK : cuda_error(e, "kv8_attention launch");
}
