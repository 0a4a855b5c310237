// Layer normalisation over the last axis and its gradient.
//
//   m = sum x / n,  r = 1 / sqrt(sum (x - m)^2 / n + eps),  h = (x - m) r,  y = h w + b
//   a = dy w,  dx = r (a - mean(a) - h mean(a h)),  dw = sum_rows dy h,  db = sum_rows dy
//
// Means, variances and all sums are float (double for float64 data); every result is rounded once.
// The variance is the mean of squared deviations from the mean (two sweeps over the row), not
// E[x^2] - m^2, which loses all digits of rows far from zero.  Every term is divided by n as it is added
// (one multiplication, fused where it can be), so that a sum overflows only where the mean itself does.
#include "row_ops.cuh"

namespace dpb {

constexpr int kThreads = 256;

// One block per row, the row read three times (the second and third time from L1/L2).
template <class T, class W>
__global__ void __launch_bounds__(kThreads) layer_norm_kernel(const T *x, RowMap xm, const W *w, const W *b, acc_t<T> eps,
                                                              T *y, RowMap ym, acc_t<T> *mean, acc_t<T> *rstd, int64_t n)
{
    using A = acc_t<T>;
    __shared__ A buf[2][kThreads / 32];
    const uint32_t r = blockIdx.x;
    const T *xr = x + xm(r);
    T *yr = y + ym(r);
    const A inv_n = A(1) / A(n);
    A s = 0;
    for (int64_t c = threadIdx.x; c < n; c += kThreads) s = fma_(to_acc<A>(xr[c]), inv_n, s);
    const A m = block_fold(SumF(), s, buf[0]);
    s = 0;
    for (int64_t c = threadIdx.x; c < n; c += kThreads) {
        const A d = to_acc<A>(xr[c]) - m;
        s = fma_(d * inv_n, d, s);
    }
    const A rs = A(1) / sqrt_(block_fold(SumF(), s, buf[1]) + eps);
    for (int64_t c = threadIdx.x; c < n; c += kThreads) {
        A h = (to_acc<A>(xr[c]) - m) * rs;
        if (w) h *= to_acc<A>(w[c]);
        if (b) h += to_acc<A>(b[c]);
        yr[c] = from_acc<T>(h);
    }
    if (threadIdx.x == 0) {
        if (mean) mean[r] = m;
        if (rstd) rstd[r] = rs;
    }
}

// Partial sums over a slab of rows: part[slab][0][c] = sum dy h, part[slab][1][c] = sum dy.
template <class T>
__global__ void __launch_bounds__(kThreads) layer_norm_columns_kernel(const T *dy, RowMap dym, const T *x, RowMap xm,
                                                                      const acc_t<T> *mean, const acc_t<T> *rstd,
                                                                      acc_t<T> *part, int64_t rows, int64_t n, int64_t slab)
{
    using A = acc_t<T>;
    const int64_t c = int64_t(blockIdx.x) * kThreads + threadIdx.x;
    if (c >= n) return;
    const int64_t first = int64_t(blockIdx.y) * slab, last = min(rows, first + slab);
    A dw = 0, db = 0;
    for (int64_t r = first; r < last; ++r) {
        const A g = to_acc<A>(dy[dym(uint32_t(r)) + c]);
        const A h = (to_acc<A>(x[xm(uint32_t(r)) + c]) - mean[r]) * rstd[r];
        dw = fma_(g, h, dw);
        db += g;
    }
    part[(int64_t(blockIdx.y) * 2) * n + c] = dw;
    part[(int64_t(blockIdx.y) * 2 + 1) * n + c] = db;
}

// dw, db = sum of the slabs in order
template <class A, class W>
__global__ void __launch_bounds__(kThreads) layer_norm_join_kernel(const A *part, int64_t slabs, int64_t n, W *dw, W *db)
{
    const int64_t i = int64_t(blockIdx.x) * kThreads + threadIdx.x;
    if (i >= 2 * n) return;
    A s = 0;
    for (int64_t k = 0; k < slabs; ++k) s += part[k * 2 * n + i];
    if (i < n) dw[i] = from_acc<W>(s);
    else db[i - n] = from_acc<W>(s);
}

template <class T, class W>
__global__ void __launch_bounds__(kThreads) layer_norm_dx_kernel(const T *dy, RowMap dym, const T *x, RowMap xm,
                                                                 const acc_t<T> *mean, const acc_t<T> *rstd, const W *w,
                                                                 T *dx, RowMap dxm, int64_t n)
{
    using A = acc_t<T>;
    __shared__ A buf[2][kThreads / 32];
    const uint32_t r = blockIdx.x;
    const T *gr = dy + dym(r), *xr = x + xm(r);
    T *o = dx + dxm(r);
    const A m = mean[r], rs = rstd[r], inv_n = A(1) / A(n);
    A s1 = 0, s2 = 0;
    for (int64_t c = threadIdx.x; c < n; c += kThreads) {
        A a = to_acc<A>(gr[c]);
        if (w) a *= to_acc<A>(w[c]);
        s1 = fma_(a, inv_n, s1);
        s2 = fma_(a * inv_n, (to_acc<A>(xr[c]) - m) * rs, s2);
    }
    const A c1 = block_fold(SumF(), s1, buf[0]);
    const A c2 = block_fold(SumF(), s2, buf[1]);
    for (int64_t c = threadIdx.x; c < n; c += kThreads) {
        A a = to_acc<A>(gr[c]);
        if (w) a *= to_acc<A>(w[c]);
        const A h = (to_acc<A>(xr[c]) - m) * rs;
        o[c] = from_acc<T>(rs * (a - c1 - h * c2));
    }
}

// --------------------------------------------------------------------------------------- launchers
struct NormArgs {
    const dpb_array *x, *w, *b, *y, *mean, *rstd;
    RowMap xm, ym;
    int64_t rows, n;
    double eps;
};

template <class T, class W> static int run_forward(const NormArgs &a, cudaStream_t s)
{
    using A = acc_t<T>;
    layer_norm_kernel<T, W><<<static_cast<unsigned>(a.rows), kThreads, 0, s>>>(
        static_cast<const T *>(a.x->data), a.xm, a.w ? static_cast<const W *>(a.w->data) : nullptr,
        a.b ? static_cast<const W *>(a.b->data) : nullptr, A(a.eps), static_cast<T *>(a.y->data), a.ym,
        a.mean ? static_cast<A *>(a.mean->data) : nullptr, a.rstd ? static_cast<A *>(a.rstd->data) : nullptr, a.n);
    note_kernel("layer_norm");
    return check_launch("layer_norm");
}

struct NormGradArgs {
    const dpb_array *dy, *x, *mean, *rstd, *w, *dx, *dw, *db;
    RowMap dym, xm, dxm;
    int64_t rows, n;
};

template <class T, class W> static int run_backward(const NormGradArgs &a, cudaStream_t s)
{
    using A = acc_t<T>;
    const T *dy = static_cast<const T *>(a.dy->data), *x = static_cast<const T *>(a.x->data);
    const A *mean = static_cast<const A *>(a.mean->data), *rstd = static_cast<const A *>(a.rstd->data);
    if (a.dw) {
        // before dx, which may overwrite dy or x
        const int64_t slabs = std::max<int64_t>(1, std::min<int64_t>(ceil_div(a.rows, 32), 64));
        const int64_t slab = std::max<int64_t>(1, ceil_div(a.rows, slabs));
        void *part = nullptr;
        DPB_TRY(dpb_malloc(static_cast<size_t>(slabs * 2 * a.n) * sizeof(A), s, &part));
        const dim3 grid(static_cast<unsigned>(ceil_div(a.n, kThreads)), static_cast<unsigned>(slabs));
        layer_norm_columns_kernel<T><<<grid, kThreads, 0, s>>>(dy, a.dym, x, a.xm, mean, rstd, static_cast<A *>(part),
                                                               a.rows, a.n, slab);
        note_kernel("layer_norm_columns");
        layer_norm_join_kernel<A, W><<<static_cast<unsigned>(ceil_div(2 * a.n, kThreads)), kThreads, 0, s>>>(
            static_cast<const A *>(part), slabs, a.n, static_cast<W *>(a.dw->data), static_cast<W *>(a.db->data));
        note_kernel("layer_norm_join");
        const int st = check_launch("layer_norm_columns");
        dpb_free(part, s);
        DPB_TRY(st);
    }
    if (a.rows == 0) return DPB_OK;
    layer_norm_dx_kernel<T, W><<<static_cast<unsigned>(a.rows), kThreads, 0, s>>>(
        dy, a.dym, x, a.xm, mean, rstd, a.w ? static_cast<const W *>(a.w->data) : nullptr,
        static_cast<T *>(a.dx->data), a.dxm, a.n);
    note_kernel("layer_norm_dx");
    return check_launch("layer_norm_dx");
}

static int check_weight(const dpb_array *w, const dpb_array &x, int wtype, const char *what)
{
    if (!w) return DPB_OK;
    DPB_TRY(check_operand(w, what));
    DPB_TRY(check_same_device(x, *w));
    DPB_TRY(check_shape(*w, nullptr, 0, x.shape[x.nd - 1], what));
    DPB_TRY(check_type(*w, wtype, what));
    DPB_TRY(check_c_contiguous(*w, what));
    if (w->typenum != x.typenum && !(x.typenum == DPB_HALF && w->typenum == DPB_FLOAT))
        return set_error(DPB_ERR_TYPE, "%s: type %s does not go with %s data", what, type_name(w->typenum),
                         type_name(x.typenum));
    return DPB_OK;
}

static int check_stat(const dpb_array *a, const dpb_array &x, const char *what)
{
    if (!a) return DPB_OK;
    DPB_TRY(check_operand(a, what));
    DPB_TRY(check_same_device(x, *a));
    DPB_TRY(check_type(*a, acc_typenum(x.typenum), what));
    DPB_TRY(check_shape(*a, x.shape, x.nd - 1, -1, what));
    return check_c_contiguous(*a, what);
}

static int check_rows(const dpb_array &x, int64_t &rows, int64_t &n)
{
    DPB_TRY(check_float_type(x, "x"));
    if (x.nd < 1) return set_error(DPB_ERR_VALUE, "x: an array of at least one dimension is needed");
    rows = count_rows(x);
    n = x.shape[x.nd - 1];
    if (n == 0) return set_error(DPB_ERR_VALUE, "normalization cannot be performed over zero-size axes");
    if (rows > kMaxRows) return set_error(DPB_ERR_VALUE, "more than 2^31 - 1 rows are not supported");
    return DPB_OK;
}

}  // namespace dpb

using namespace dpb;

extern "C" {

int dpb_layer_norm(const dpb_array *x, const dpb_array *weight, const dpb_array *bias, double eps, const dpb_array *y,
                   const dpb_array *mean, const dpb_array *rstd, void *stream)
{
    DPB_TRY(check_operand(x, "x"));
    DPB_TRY(check_operand(y, "y"));
    NormArgs a = {};
    DPB_TRY(check_rows(*x, a.rows, a.n));
    if (!(eps >= 0) || std::isinf(eps)) return set_error(DPB_ERR_VALUE, "eps must be a finite number that is not negative");
    const int wt = weight ? weight->typenum : bias ? bias->typenum : x->typenum;
    DPB_TRY(check_weight(weight, *x, wt, "weight"));
    DPB_TRY(check_weight(bias, *x, wt, "bias"));
    DPB_TRY(check_same_device(*x, *y));
    DPB_TRY(check_type(*y, x->typenum, "y"));
    DPB_TRY(check_shape(*y, x->shape, x->nd, -1, "y"));
    DPB_TRY(check_stat(mean, *x, "mean"));
    DPB_TRY(check_stat(rstd, *x, "rstd"));
    for (const dpb_array *o : {y, mean, rstd})
        if (o) DPB_TRY(check_output(*o, "output"));
    if (a.rows == 0) return DPB_OK;
    DPB_TRY(check_row_map(*x, a.xm, "x"));
    DPB_TRY(check_row_map(*y, a.ym, "y"));
    DPB_TRY(check_no_overlap(*x, *y, true));
    DPB_TRY(check_no_overlaps({x}, {mean, rstd}));
    DPB_TRY(check_no_overlaps({weight, bias}, {y, mean, rstd}));
    a.x = x, a.w = weight, a.b = bias, a.y = y, a.mean = mean, a.rstd = rstd, a.eps = eps;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (x->typenum == DPB_DOUBLE) return run_forward<double, double>(a, s);
    if (x->typenum == DPB_FLOAT) return run_forward<float, float>(a, s);
    return wt == DPB_FLOAT ? run_forward<half_t, float>(a, s) : run_forward<half_t, half_t>(a, s);
}

int dpb_layer_norm_backward(const dpb_array *dy, const dpb_array *x, const dpb_array *mean, const dpb_array *rstd,
                            const dpb_array *weight, const dpb_array *dx, const dpb_array *dweight,
                            const dpb_array *dbias, void *stream)
{
    DPB_TRY(check_operand(x, "x"));
    DPB_TRY(check_operand(dy, "dy"));
    DPB_TRY(check_operand(dx, "dx"));
    NormGradArgs a = {};
    DPB_TRY(check_rows(*x, a.rows, a.n));
    if (!mean || !rstd) return set_error(DPB_ERR_VALUE, "mean and rstd are needed");
    if (!dweight != !dbias) return set_error(DPB_ERR_VALUE, "dweight and dbias come together");
    const int wt = weight ? weight->typenum : dweight ? dweight->typenum : x->typenum;
    DPB_TRY(check_weight(weight, *x, wt, "weight"));
    DPB_TRY(check_weight(dweight, *x, wt, "dweight"));
    DPB_TRY(check_weight(dbias, *x, wt, "dbias"));
    for (const dpb_array *o : {dy, dx}) {
        DPB_TRY(check_same_device(*x, *o));
        DPB_TRY(check_type(*o, x->typenum, o == dy ? "dy" : "dx"));
        DPB_TRY(check_shape(*o, x->shape, x->nd, -1, o == dy ? "dy" : "dx"));
    }
    DPB_TRY(check_stat(mean, *x, "mean"));
    DPB_TRY(check_stat(rstd, *x, "rstd"));
    for (const dpb_array *o : {dx, dweight, dbias})
        if (o) DPB_TRY(check_output(*o, "output"));
    if (a.rows > 0) {
        DPB_TRY(check_row_map(*x, a.xm, "x"));
        DPB_TRY(check_row_map(*dy, a.dym, "dy"));
        DPB_TRY(check_row_map(*dx, a.dxm, "dx"));
    }
    DPB_TRY(check_no_overlap(*x, *dx, true));
    DPB_TRY(check_no_overlap(*dy, *dx, true));
    DPB_TRY(check_no_overlaps({x, dy}, {dweight, dbias}));
    DPB_TRY(check_no_overlaps({mean, rstd, weight}, {dx, dweight, dbias}));
    a.dy = dy, a.x = x, a.mean = mean, a.rstd = rstd, a.w = weight, a.dx = dx, a.dw = dweight, a.db = dbias;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (x->typenum == DPB_DOUBLE) return run_backward<double, double>(a, s);
    if (x->typenum == DPB_FLOAT) return run_backward<float, float>(a, s);
    return wt == DPB_FLOAT ? run_backward<half_t, float>(a, s) : run_backward<half_t, half_t>(a, s);
}

}  // extern "C"
