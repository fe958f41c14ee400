// C entry points of the root-mean-square norm and of rotary positions (include/fss_b200.h).
#include "fss_host.cuh"
#include "fss_norm.cuh"
#include "fss_rotary.cuh"

namespace fss {
namespace {

template <typename T> bool wide_view(const fss_view *v, int64_t B, int64_t Tn) {
    constexpr int64_t V = VecWidth<T>::value;
    return !v || !v->ptr || (aligned16(v->ptr) && (Tn <= 1 || v->stride_t % V == 0) && (B <= 1 || v->stride_b % V == 0));
}

// Whether the rows of a tensor lie evenly, from one sequence to the next.
inline bool even(const fss_view *v, int64_t B, int64_t Tn) { return !v || !v->ptr || B <= 1 || v->stride_b == Tn * v->stride_t; }

// How a row is laid over threads: fragments a thread and threads a row.  Up to 4 fragments for each lane of a warp, a
// warp takes a row by itself; else a CTA does, with as few fragments a thread as it has threads for.
struct Layout { int fragments, threads; bool block; };
inline Layout choose_layout(int64_t n) {      // n: fragments of a row; threads 0: too many
    if (n <= 32) return {1, 256, false};
    if (n <= 64) return {2, 256, false};
    if (n <= 128) return {4, 256, false};
    for (int f : {1, 2, 4})
        if (n <= f * 512 || (f == 4 && n <= f * 1024)) return {f, (int)(ceil_div(ceil_div(n, f), 32) * 32), true};
    return {0, 0, true};
}

template <typename T, int kQuant> int norm_forward(const norm::Params<T> &p, bool vec, bool wide, cudaStream_t stream) {
    constexpr int V = VecWidth<T>::value;
    const int64_t rows = p.B * p.T_;
    const Layout w = vec ? choose_layout(p.D / V) : Layout{0, 0, true};
    if (w.threads == 0) {
        norm::forward_any<T, kQuant><<<(unsigned)rows, 256, 0, stream>>>(p, wide);
        return launch_check("norm launch");
    }
    const unsigned blocks = (unsigned)(w.block ? rows : ceil_div(rows, w.threads / 32));
#define FSS_NORM(N, BLOCK) norm::forward<T, N, BLOCK, kQuant><<<blocks, w.threads, 0, stream>>>(p, wide)
    if (w.block) {
        if (w.fragments == 1) FSS_NORM(1, true);
        else if (w.fragments == 2) FSS_NORM(2, true);
        else FSS_NORM(4, true);
    } else {
        if (w.fragments == 1) FSS_NORM(1, false);
        else if (w.fragments == 2) FSS_NORM(2, false);
        else FSS_NORM(4, false);
    }
#undef FSS_NORM
    return launch_check("norm launch");
}

template <typename T>
int run_norm(const fss_scan_ctx *ctx, int64_t B, int64_t Tn, int64_t D, const fss_view *x, const fss_view *residual, const fss_norm_weight *weight, float eps,
             const fss_view *sum, const fss_norm_output *out) {
    norm::Params<T> p{};
    p.B = B; p.T_ = Tn; p.D = D;
    p.x = make_view<const T>(x);
    if (residual) { p.residual = make_view<const T>(residual); p.sum = make_view<T>(sum); }
    if (out->y.ptr) p.y = make_view<T>(&out->y);
    p.held = static_cast<__nv_fp8_e4m3 *>(out->held);
    p.scales = out->scales;
    p.rstd = out->rstd;
    p.weight = weight->ptr;
    p.eps = eps;
    p.group = out->group;
    if (even(x, B, Tn) && even(residual, B, Tn) && even(residual ? sum : nullptr, B, Tn) && even(&out->y, B, Tn)) { p.B = 1; p.T_ = B * Tn; }
    const bool wide = weight->dtype == FSS_DTYPE_F32;
    const bool vec = D % VecWidth<T>::value == 0 && wide_view<T>(x, B, Tn) && wide_view<T>(residual, B, Tn) && wide_view<T>(residual ? sum : nullptr, B, Tn) &&
                     wide_view<T>(&out->y, B, Tn) && aligned16(weight->ptr) && aligned16(out->held);
    cudaStream_t stream = (cudaStream_t)ctx->stream;
    if (!out->held) return norm_forward<T, norm::kNone>(p, vec, wide, stream);
    if (!out->group) return norm_forward<T, norm::kRow>(p, vec, wide, stream);
    return norm_forward<T, norm::kGroup>(p, vec, wide, stream);
}

constexpr int kNormWalkers = 148 * 8;      // rows of partial sums at most; also how many walkers fill the device

template <typename T>
int run_norm_backward(const fss_scan_ctx *ctx, int64_t B, int64_t Tn, int64_t D, const fss_view *s, const fss_norm_weight *weight, const float *rstd,
                      const fss_view *dy, const fss_view *dsum, const fss_view *dx, void *dweight) {
    constexpr int V = VecWidth<T>::value;
    norm::BackwardParams<T> p{};
    p.B = B; p.T_ = Tn; p.D = D;
    p.s = make_view<const T>(s);
    p.dy = make_view<const T>(dy);
    if (dsum) p.dsum = make_view<const T>(dsum);
    p.dx = make_view<T>(dx);
    p.rstd = rstd;
    p.weight = weight->ptr;
    p.parts = dweight ? static_cast<float *>(ctx->workspace) : nullptr;
    if (even(s, B, Tn) && even(dy, B, Tn) && even(dsum, B, Tn) && even(dx, B, Tn)) { p.B = 1; p.T_ = B * Tn; }
    const bool wide = weight->dtype == FSS_DTYPE_F32;
    const bool vec = D % V == 0 && wide_view<T>(s, B, Tn) && wide_view<T>(dy, B, Tn) && wide_view<T>(dsum, B, Tn) && wide_view<T>(dx, B, Tn) && aligned16(weight->ptr);
    cudaStream_t stream = (cudaStream_t)ctx->stream;
    const int64_t rows = B * Tn;
    const Layout w = vec ? choose_layout(D / V) : Layout{0, 0, true};
    int64_t parts;
    if (w.threads == 0) {
        parts = rows < 148 * 4 ? rows : 148 * 4;
        norm::backward_any<T><<<(unsigned)parts, 256, 0, stream>>>(p, wide);
    } else {
        const int per = w.block ? 1 : w.threads / 32;
        int64_t blocks = ceil_div(rows, per);
        const int64_t most = w.block ? 148 * (1024 / w.threads > 1 ? 1024 / w.threads : 1) : kNormWalkers / per;
        if (blocks > most) blocks = most;
        parts = blocks * per < rows ? blocks * per : rows;
#define FSS_NORM(N, BLOCK) norm::backward<T, N, BLOCK><<<(unsigned)blocks, w.threads, 0, stream>>>(p, wide)
        if (w.block) {
            if (w.fragments == 1) FSS_NORM(1, true);
            else if (w.fragments == 2) FSS_NORM(2, true);
            else FSS_NORM(4, true);
        } else {
            if (w.fragments == 1) FSS_NORM(1, false);
            else if (w.fragments == 2) FSS_NORM(2, false);
            else FSS_NORM(4, false);
        }
#undef FSS_NORM
    }
    if (dweight) norm::sum_parts<<<(unsigned)ceil_div(D, 32), 256, 0, stream>>>(p.parts, parts, D, dweight, wide);
    return launch_check("norm gradient launch");
}

int check_rows(int dtype, int64_t B, int64_t Tn, int64_t D) {
    if (dtype != FSS_DTYPE_BF16 && dtype != FSS_DTYPE_F32) return FSS_E_DTYPE;
    if (B < 0 || Tn < 0 || D < 1) return FSS_E_SHAPE;
    if (B > 0 && Tn > INT32_MAX / B) return FSS_E_SHAPE;      // rows are numbered by the grid
    if (B * Tn > 0 && D > (INT64_MAX / 32) / (B * Tn)) return FSS_E_SHAPE;
    return FSS_OK;
}
int check_weight(const fss_norm_weight *w, int dtype) {
    if (!w || !w->ptr) return FSS_E_NULL;
    return w->dtype == dtype || w->dtype == FSS_DTYPE_F32 ? FSS_OK : FSS_E_DTYPE;
}

// ------------------------------------------------------------------ rotary positions
template <typename T> bool wide_side(const fss_heads *x, int64_t B, int64_t Tn, int V) {
    const int64_t n = V;
    return reinterpret_cast<uintptr_t>(x->ptr) % (n * sizeof(T)) == 0 && (B <= 1 || x->stride_b % n == 0) && (Tn <= 1 || x->stride_t % n == 0) &&
           (x->heads <= 1 || x->stride_h % n == 0);
}

template <typename T>
int run_rotary(const fss_scan_ctx *ctx, int64_t B, int64_t Tn, const fss_heads *const (&in)[2], void *const (&out)[2], const fss_rotary *r) {
    constexpr int V = VecWidth<T>::value;
    rotary::Params<T> p{};
    p.B = B; p.T_ = Tn;
    p.D = (int)in[0]->dim;
    p.R = (int)r->rotary_dim;
    bool vec = p.D % V == 0 && (r->interleaved ? p.R % V == 0 : p.R / 2 % V == 0);
    int64_t heads = 0;
    for (int i = 0; i < 2; ++i) {
        if (!in[i]) continue;
        p.side[i] = {static_cast<const T *>(in[i]->ptr), in[i]->stride_b, in[i]->stride_t, in[i]->stride_h, static_cast<T *>(out[i]), (int)in[i]->heads};
        vec = vec && wide_side<T>(in[i], B, Tn, V) && aligned16(out[i]);
        heads += in[i]->heads;
    }
    p.positions = r->positions;
    p.psb = r->position_stride_b; p.pst = r->position_stride_t;
    p.turns = r->turns;
    p.magnitude = r->magnitude;
    const int64_t rows = B * Tn, per_head = vec ? (r->interleaved ? p.D / V : (p.D - p.R / 2) / V) : p.D - p.R / 2, per_token = heads * per_head;
    // about 4,096 items a CTA, and no more than 4,096 sines and kMaxTokens tokens; a few tokens are shared by several CTAs instead
    int64_t tokens = 4096 / per_token, most = 4096 / (p.R / 2);
    if (tokens > most) tokens = most;
    if (tokens > rotary::kMaxTokens) tokens = rotary::kMaxTokens;
    if (tokens > rows / (4 * 148)) tokens = rows / (4 * 148);
    p.tokens = (int)(tokens < 1 ? 1 : tokens);
    const int64_t groups = ceil_div(rows, p.tokens);
    int64_t splits = groups >= 148 ? 1 : ceil_div(148, groups), useful = ceil_div(p.tokens * per_token, rotary::kThreads);
    p.splits = (int)(splits < useful ? splits : useful);
    if (groups * p.splits > INT32_MAX) return FSS_E_SHAPE;
    const unsigned blocks = (unsigned)(groups * p.splits);
    const size_t smem = (size_t)p.tokens * (p.R / 2) * sizeof(float2);
    cudaStream_t stream = (cudaStream_t)ctx->stream;
    void (*kernel)(rotary::Params<T>);
    if (vec) {
        if (r->interleaved) kernel = r->inverse ? rotary::rotate<T, V, true, true> : rotary::rotate<T, V, true, false>;
        else kernel = r->inverse ? rotary::rotate<T, V, false, true> : rotary::rotate<T, V, false, false>;
    } else {
        if (r->interleaved) kernel = r->inverse ? rotary::rotate<T, 1, true, true> : rotary::rotate<T, 1, true, false>;
        else kernel = r->inverse ? rotary::rotate<T, 1, false, true> : rotary::rotate<T, 1, false, false>;
    }
    kernel<<<blocks, rotary::kThreads, smem, stream>>>(p);
    return launch_check("rotary launch");
}

}  // namespace
}  // namespace fss

using namespace fss;

FSS_API int fss_rms_norm_forward(const fss_scan_ctx *ctx, int dtype, int64_t B, int64_t T, int64_t D, const fss_view *x, const fss_view *residual,
                                 const fss_norm_weight *weight, float eps, const fss_view *sum, const fss_norm_output *out) {
    int rc;
    if ((rc = check_ctx(ctx)) || (rc = check_rows(dtype, B, T, D)) || (rc = check_weight(weight, dtype))) return rc;
    if (!out || (!out->y.ptr && !out->held)) return FSS_E_NULL;
    if (residual && !sum) return FSS_E_NULL;
    if (out->y.ptr && out->held) return FSS_E_ARGS;
    if (out->held && (!out->scales || (out->group != 0 && out->group != 32 && out->group != 64 && out->group != 128) || (out->group && D % out->group))) return FSS_E_ARGS;
    if (B * T == 0) return FSS_OK;
    if ((rc = check_view_extents(x, B, T, D)) || (residual && ((rc = check_view_extents(residual, B, T, D)) || (rc = check_view_extents(sum, B, T, D)))) ||
        (out->y.ptr && (rc = check_view_extents(&out->y, B, T, D))))
        return rc;
    DeviceGuard guard(ctx->device);
    if (guard.error) return guard.error;
    return dtype == FSS_DTYPE_BF16 ? run_norm<bf16>(ctx, B, T, D, x, residual, weight, eps, sum, out)
                                   : run_norm<float>(ctx, B, T, D, x, residual, weight, eps, sum, out);
}

FSS_API size_t fss_rms_norm_workspace_bytes(int64_t D) { return D > 0 ? (size_t)kNormWalkers * (size_t)D * sizeof(float) : 0; }

FSS_API int fss_rms_norm_backward(const fss_scan_ctx *ctx, int dtype, int64_t B, int64_t T, int64_t D, const fss_view *s, const fss_norm_weight *weight,
                                  const float *rstd, const fss_view *dy, const fss_view *dsum, const fss_view *dx, void *dweight) {
    int rc;
    if ((rc = check_ctx(ctx)) || (rc = check_rows(dtype, B, T, D)) || (rc = check_weight(weight, dtype))) return rc;
    if (B * T == 0) return FSS_OK;
    if (!rstd) return FSS_E_NULL;
    if ((rc = check_view_extents(s, B, T, D)) || (rc = check_view_extents(dy, B, T, D)) || (dsum && (rc = check_view_extents(dsum, B, T, D))) ||
        (rc = check_view_extents(dx, B, T, D)))
        return rc;
    if (dweight && (!ctx->workspace || ctx->workspace_bytes < fss_rms_norm_workspace_bytes(D))) return FSS_E_WORKSPACE;
    DeviceGuard guard(ctx->device);
    if (guard.error) return guard.error;
    return dtype == FSS_DTYPE_BF16 ? run_norm_backward<bf16>(ctx, B, T, D, s, weight, rstd, dy, dsum, dx, dweight)
                                   : run_norm_backward<float>(ctx, B, T, D, s, weight, rstd, dy, dsum, dx, dweight);
}

FSS_API int fss_rotary_apply(const fss_scan_ctx *ctx, int dtype, int64_t B, int64_t T, const fss_heads *q, const fss_heads *k, void *q_out, void *k_out,
                             const fss_rotary *r) {
    int rc;
    if ((rc = check_ctx(ctx))) return rc;
    if (!q || !r || (k && !k_out)) return FSS_E_NULL;
    if (r->struct_bytes != sizeof(fss_rotary)) return FSS_E_ARGS;
    if (dtype != FSS_DTYPE_BF16 && dtype != FSS_DTYPE_F32) return FSS_E_DTYPE;
    if (B < 0 || T < 0 || r->rotary_dim < 2 || r->rotary_dim % 2 || r->rotary_dim > q->dim || (k && k->dim != q->dim)) return FSS_E_SHAPE;
    if (r->rotary_dim > 2 * rotary::kMaxPairs || q->dim > 65536 || q->heads > 65536 || (k && k->heads > 65536)) return FSS_E_TOO_LARGE;
    if (B > 0 && T > INT32_MAX / B) return FSS_E_SHAPE;
    for (const fss_heads *x : {q, k})
        if (x && (x->heads < 1 || x->stride_b < 0 || x->stride_t < 0 || x->stride_h < 0 || (B > 1 && x->stride_b > (INT64_MAX / 32) / B) ||
                  (T > 1 && x->stride_t > (INT64_MAX / 32) / T)))
            return FSS_E_SHAPE;
    if ((q->heads + (k ? k->heads : 0)) * q->dim > (1 << 26)) return FSS_E_TOO_LARGE;
    if (B * T == 0) return FSS_OK;
    if (!q->ptr || !q_out || (k && !k->ptr) || !r->positions || !r->turns) return FSS_E_NULL;
    DeviceGuard guard(ctx->device);
    if (guard.error) return guard.error;
    const fss_heads *const in[2] = {q, k};
    void *const out[2] = {q_out, k_out};
    return dtype == FSS_DTYPE_BF16 ? run_rotary<bf16>(ctx, B, T, in, out, r) : run_rotary<float>(ctx, B, T, in, out, r);
}
