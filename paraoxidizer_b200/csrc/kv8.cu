// kv8.cu -- the 8-bit paged KV cache next to the decode path: norms and rotation of q and k rows,
// appending k and v rows to int8 pages, reading rows back, and the entry points of include/pox_cuda.h
// (the attention's kernels are in kv8_attn.cu).
#include <algorithm>
#include <new>

#include "../../include/pox_cuda.h"
#include "api_internal.h"
#include "kv8.cuh"
#include "kv8_attn.h"

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

// One warp per (row, head): a pass for the sum of squares, one for the pairs.
template <typename T>
__global__ void __launch_bounds__(256) qk_norm_rope_kernel(QkArgs<T> a) {
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

// ---- append ----------------------------------------------------------------------------------------
template <typename T>
struct AppendArgs {
    Kv8Cache c;
    Kv8Batch b;
    RowsView<const T> x[2];
    RopeView rope;
    int* err;
};

// A page of the batch: sequence s owns page items (row_starts[s] + 30 s) / 16 .. (a bound of the pages that
// its n rows touch: n rows reach at most (n + 30) / 16 pages, in closed form, so no scan over the sequences).
__device__ __forceinline__ uint32_t page_base(const Kv8Batch& b, uint32_t s) {
    return b.max_rows == 1 && !b.row_starts ? s : (uint32_t)(((unsigned long long)b.row_starts[s] + 30ull * s) / 16);
}

// One warp per (touched page, kv head, side): the page's new rows set the scale, its older slots follow.
template <int HD, typename T>
__global__ void __launch_bounds__(128) kv8_append_kernel(AppendArgs<T> a, uint32_t items) {
    const int lane = threadIdx.x & 31, E = HD / 32;
    const unsigned long long u = (unsigned long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    const uint32_t item = (uint32_t)(u / (2 * a.c.kvh));
    const int side = (int)(u % 2), h = (int)(u / 2 % a.c.kvh);
    if (item >= items) return;
    const uint32_t s = a.b.row_starts ? find_seq(a.b, item, 30, 16) : item;
    SeqSpan sp;
    if (!seq_span(a.b, s, sp, a.err)) return;
    const int p0 = max(sp.ctx - sp.n, 0), page = p0 / kPage + (int)(item - page_base(a.b, s));
    if (sp.ctx <= p0 || page * kPage >= sp.ctx) return;
    const int first = max(p0 - page * kPage, 0), last = min(sp.ctx - page * kPage, kPage);
    const int blk = a.b.btab[(size_t)s * a.b.mbps + page];
    if (blk < 0 || (uint32_t)blk >= a.c.num_blocks) {
        if (lane == 0) atomicOr(a.err, kErrAttnPage);
        return;
    }
    const int rot = a.rope.rot, half = rot / 2;
    if (side == 0 && rot && (uint32_t)(page * kPage + last - 1) >= a.rope.positions) {
        if (lane == 0) atomicOr(a.err, kErrRopePos);
        return;
    }
    int8_t* pg = a.c.pages + ((size_t)blk * a.c.kvh + h) * (2 * kPage * HD);
    float* sc = a.c.scales + ((size_t)blk * a.c.kvh + h) * 2 + side;
    auto elem = [&](int t, int d) {  // the row element that slot t stores
        const int pos = page * kPage + t;
        const T* x = a.x[side].at((size_t)sp.r0 + (pos - (sp.ctx - sp.n)), h);
        float v = to_f32(x[d]);
        if (side == 0 && d < rot) {
            const bool low = a.rope.half ? d < half : !(d & 1);
            const int o = a.rope.half ? (low ? d + half : d - half) : d ^ 1, i = a.rope.half ? (low ? d : o) : d / 2;
            const float w = to_f32(x[o]);
            const float2 r = rope_turn(low ? v : w, low ? w : v, a.rope.table[(size_t)pos * half + i]);
            v = low ? r.x : r.y;
        }
        return v;
    };
    float m = 0.f;
    for (int t = first; t < last; t++)
        for (int e = 0; e < E; e++) {
            const float v = fabsf(elem(t, lane + 32 * e));
            if (v < INFINITY) m = fmaxf(m, v);  // false for NaN too
        }
    m = warp_max(m);
    const float old = first ? *sc : 0.f;
    const float now = fmaxf(old, __fdiv_rn(m, 127.f));
    const float ratio = now > 0.f ? __fdiv_rn(old, now) : 0.f;
    auto put = [&](int t, int d) -> int8_t& { return pg[side ? kv8_v_off<HD>(t, d) : kv8_k_off<HD>(t, d)]; };
    for (int e = 0; e < E; e++) {
        const int d = lane + 32 * e;
        for (int t = 0; t < first; t++) put(t, d) = (int8_t)__float2int_rn(__fmul_rn((float)put(t, d), ratio));
        for (int t = first; t < last; t++) {
            const float q = now > 0.f ? __fdiv_rn(elem(t, d), now) : 0.f;
            put(t, d) = (int8_t)__float2int_rn(fminf(fmaxf(q, -127.f), 127.f) * (q == q ? 1.f : 0.f));
        }
    }
    __syncwarp();
    if (lane == 0) *sc = now;
}

// ---- reading rows back -------------------------------------------------------------------------------
template <int HD, typename T>
__global__ void __launch_bounds__(128) kv8_read_kernel(Kv8Cache c, Kv8Batch b, RowsView<T> k, RowsView<T> v, int* err) {
    const int lane = threadIdx.x & 31;
    const unsigned long long u = (unsigned long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    const uint32_t r = (uint32_t)(u / c.kvh);
    const int h = (int)(u % c.kvh);
    if (r >= b.rows) return;
    const uint32_t s = b.row_starts ? find_seq(b, r, 0, 1) : r;
    SeqSpan sp;
    if (!seq_span(b, s, sp, err)) return;
    const int pos = sp.ctx - sp.n + (int)(r - sp.r0);
    const int blk = pos >= 0 ? b.btab[(size_t)s * b.mbps + pos / kPage] : 0;
    if (blk < 0 || (uint32_t)blk >= c.num_blocks) {
        if (lane == 0) atomicOr(err, kErrAttnPage);
        return;
    }
    const int8_t* pg = c.pages + ((size_t)blk * c.kvh + h) * (2 * kPage * HD);
    const float* sc = c.scales + ((size_t)blk * c.kvh + h) * 2;
    const int t = pos % kPage;
    for (int d = lane; d < HD; d += 32) {
        k.at(r, h)[d] = from_f32<T>(pos < 0 ? 0.f : (float)pg[kv8_k_off<HD>(t, d)] * sc[0]);
        v.at(r, h)[d] = from_f32<T>(pos < 0 ? 0.f : (float)pg[kv8_v_off<HD>(t, d)] * sc[1]);
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
    if (far >= ((unsigned __int128)1 << 46)) return set_error(POX_ERR_INVALID, "%s: strides out of range", what);
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
        v = RopeView{reinterpret_cast<const float2*>(r->table), r->positions, (int)r->rot_dim, r->style == POX_ROPE_HALF};
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
    return Kv8Batch{b->row_starts, b->ctx_lens, b->block_tables, b->seqs, b->rows, b->max_rows, b->max_ctx,
                    b->max_blocks_per_seq};
}

constexpr int kPromptRows = 64;

// The stream's split partials and tickets for a plan that splits.
static int kv8_scratch(pox_cuda_ctx* ctx, cudaStream_t st, uint32_t hd, Kv8StepPlan& p) {
    if (p.splits <= 1) return POX_OK;
    const size_t need = p.items * p.splits * (p.pair ? 8 : 16) * (hd + 2) * sizeof(float);
    try {
        std::lock_guard<std::mutex> lk(ctx->mu);
        Kv8Scratch& k = ctx->kv8[st];
        if (need > k.part_bytes || p.items > k.items) {
            cudaStreamCaptureStatus cs = cudaStreamCaptureStatusNone;
            if (cudaStreamIsCapturing(st, &cs) != cudaSuccess || cs != cudaStreamCaptureStatusNone)
                return set_error(POX_ERR_INVALID, "split partials must be sized by a call before stream capture");
            cudaError_t e = cudaStreamSynchronize(st);  // earlier calls may still use the old ones
            if (e != cudaSuccess) return cuda_error(e, "cudaStreamSynchronize");
            const size_t bytes = std::max(need, k.part_bytes), items = std::max(p.items, k.items);
            cudaFree(k.part);
            cudaFree(k.tickets);
            k = Kv8Scratch();
            e = cudaMalloc(&k.part, bytes);
            if (e == cudaSuccess) k.part_bytes = bytes, e = cudaMalloc(&k.tickets, items * sizeof(uint32_t));
            if (e == cudaSuccess) k.items = items, e = cudaMemsetAsync(k.tickets, 0, items * sizeof(uint32_t), st);
            if (e != cudaSuccess) {
                k.items = 0;  // so that the next call allocates and clears again
                return cuda_error(e, "split partials");
            }
        }
        p.part = k.part;
        p.tickets = k.tickets;
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
    const unsigned long long items = (unsigned long long)a->rows * (a->heads + a->kv_heads);
    qk_norm_rope_kernel<T><<<(unsigned)((items + 7) / 8), 256, 0, st>>>(k);
    return cudaGetLastError();
}

template <int HD, typename T>
static cudaError_t launch_append(pox_cuda_ctx* ctx, const pox_kv8_cache* c, const pox_kv8_batch* b, const pox_rows* k,
                                 const pox_rows* v, const pox_rope* rope, cudaStream_t st) {
    AppendArgs<T> a{cache_view(c), batch_view(b), {rows_view<const T>(*k), rows_view<const T>(*v)}, rope_view(rope),
                    ctx->err_dev};
    const uint32_t items = b->row_starts ? (uint32_t)((b->rows + 30ull * b->seqs) / 16 + 1) : b->seqs;
    const unsigned long long warps = (unsigned long long)items * c->kv_heads * 2;
    kv8_append_kernel<HD, T><<<(unsigned)((warps + 3) / 4), 128, 0, st>>>(a, items);
    return cudaGetLastError();
}

template <int HD, typename T>
static cudaError_t launch_read(pox_cuda_ctx* ctx, const pox_kv8_cache* c, const pox_kv8_batch* b, const pox_rows* k,
                               const pox_rows* v, cudaStream_t st) {
    const unsigned long long warps = (unsigned long long)b->rows * c->kv_heads;
    kv8_read_kernel<HD, T><<<(unsigned)((warps + 3) / 4), 128, 0, st>>>(cache_view(c), batch_view(b), rows_view<T>(*k),
                                                                        rows_view<T>(*v), ctx->err_dev);
    return cudaGetLastError();
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
        if (s.in->data == s.out->data && (s.in->row_stride != s.out->row_stride || s.in->head_stride != s.out->head_stride))
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

static int check_kv_rows(const pox_kv8_cache* c, const pox_kv8_batch* b, const pox_rows* k, const pox_rows* v, bool written) {
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

extern "C" int pox_cuda_kv8_attention(pox_cuda_ctx* ctx, const pox_kv8_cache* c, const pox_kv8_batch* b, const pox_rows* q,
                                      const pox_rows* out, uint32_t heads, float scale, void* stream) {
    if (!ctx) return set_error(POX_ERR_INVALID, "ctx is NULL");
    int rc = check_cache(c, b);
    if (rc || b->rows == 0 || b->seqs == 0) return rc;
    if (!heads || heads % c->kv_heads) return set_error(POX_ERR_INVALID, "%u heads over %u kv heads", heads, c->kv_heads);
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
    const int G = (int)(heads / c->kv_heads), es = esize(q->dtype);
    // Sequences of more rows than kPromptRows go to the tensor-memory kernel; a batch may hold both kinds,
    // told apart on the device. All rows equal (or one sequence) means one kind.
    const long long most = (long long)b->max_rows * G;
    const bool prompt = c->head_dim != 32 && q->dtype != POX_F32 && most > kPromptRows;
    const bool step = !prompt || (b->seqs > 1 && b->rows != (unsigned long long)b->seqs * b->max_rows);
    Kv8StepPlan plan = kv8_step_plan(batch_view(b), (int)c->kv_heads, G, q->dtype == POX_F32, ctx->num_sms,
                                     prompt ? kPromptRows : 0x7fffffff);
    if (plan.items * (unsigned __int128)plan.splits > 0x7fffffffu)
        return set_error(POX_ERR_UNSUPPORTED, "%zu items of %d splits", plan.items, plan.splits);
    plan.device = ctx->device;
    rc = step ? kv8_scratch(ctx, st, c->head_dim, plan) : POX_OK;
    if (rc) return rc;
    const int vec = (((uintptr_t)q->data | (uintptr_t)out->data) % (4 * es)) == 0 &&
                    ((q->row_stride | q->head_stride | out->row_stride | out->head_stride) % 4) == 0;
    e = by_shape(c->head_dim, q->dtype, [&](auto hd, auto t) {
        using T = decltype(t);
        const float s = (scale > 0.f ? scale : 1.0f / sqrtf((float)c->head_dim)) * 1.4426950408889634f;
        Kv8Attn<T> a{cache_view(c), batch_view(b), rows_view<const T>(*q), rows_view<T>(*out), G, s, vec, ctx->err_dev};
        constexpr int HD = decltype(hd)::value;
        cudaError_t r = cudaSuccess;
        if constexpr (HD != 32 && sizeof(T) == 2)
            if (prompt) r = launch_kv8_prompt<HD, T>(a, kPromptRows + 1, ctx->device, st);
        if (r == cudaSuccess && step) r = launch_kv8_step<HD, T>(a, plan, st);
        return r;
    });
    return e == cudaSuccess ? POX_OK : cuda_error(e, "kv8_attention launch");
}
