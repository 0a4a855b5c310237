// Distillation loss from a teacher's top logits, and its gradient.
//
// Row r has V student logits z and K teacher logits t at columns j.  An entry counts when 0 <= j < V
// and t > -inf.  With a temperature T,
//   p = softmax(t / T) over the entries that count,  q = softmax(z / T),
//   loss = T^2 sum_k p_k (log p_k - log q_{j_k}),    dz = dloss T (q - sum_{k: j_k = .} p_k).
// A row without entries (padding, a prompt) has loss 0 and gradient 0, and its logits are not read.
// Where q is 0 (z = -inf, or every z of the row) and p is not, the loss is +inf; q counts as 0 in dz.
//
// log q = (z - max z) / T - log sum exp((z - max z) / T): the differences are taken before the
// division, so that logits of the type's lowest value do not overflow.  The two statistics (max z, log
// of the sum) are kept apart for the backward pass: their sum would lose log2 |max z| bits.  All of it
// is float (double for float64 logits); each gradient is rounded once.
#include "row_ops.cuh"

namespace dpb {

constexpr int kThreads = 256;
constexpr int kMaxTop = 1024;   // teacher entries a row may have

// What a block keeps of its row's teacher: probabilities, their logarithms and columns (-1: does not count).
template <class A> struct Teacher {
    A p[kMaxTop];
    A logp[kMaxTop];
    int64_t at[kMaxTop];
};

// Fills `t` for one row; false when no entry counts.  Ends with the block synchronised.
template <class A, class I>
DPB_D bool load_teacher(Teacher<A> &t, const A *top, const I *index, int k, int64_t vocab, A inv_temp, A *buf)
{
    A best = -INFINITY;
    int any = 0;
    for (int i = threadIdx.x; i < k; i += kThreads) {
        const A v = top[i];
        const int64_t j = static_cast<int64_t>(index[i]);
        const bool counts = j >= 0 && j < vocab && !(v == -INFINITY);
        t.at[i] = counts ? j : -1;
        t.logp[i] = v;
        if (counts) {
            best = MaxF()(best, v);
            any = 1;
        }
    }
    any = __syncthreads_or(any);
    if (!any) return false;
    best = block_fold(MaxF(), best, buf);
    __syncthreads();
    A sum = 0;
    for (int i = threadIdx.x; i < k; i += kThreads) {
        const A e = t.at[i] >= 0 ? exp_((t.logp[i] - best) * inv_temp) : A(0);
        t.p[i] = e;
        sum += e;
    }
    sum = block_fold(SumF(), sum, buf);
    const A log_sum = log_(sum);
    for (int i = threadIdx.x; i < k; i += kThreads) {
        t.p[i] = t.p[i] / sum;
        t.logp[i] = t.at[i] >= 0 ? (t.logp[i] - best) * inv_temp - log_sum : A(0);
    }
    __syncthreads();
    return true;
}

template <class T, class I>
__global__ void __launch_bounds__(kThreads) distillation_loss_kernel(const T *z, RowMap zm, const acc_t<T> *top, const I *index,
                                                                     int k, int64_t vocab, acc_t<T> temp, acc_t<T> inv_temp,
                                                                     acc_t<T> *loss, acc_t<T> *stats)
{
    using A = acc_t<T>;
    __shared__ Teacher<A> t;
    __shared__ A buf[kThreads / 32];
    const uint32_t r = blockIdx.x;
    if (!load_teacher(t, top + int64_t(r) * k, index + int64_t(r) * k, k, vocab, inv_temp, buf)) {
        if (threadIdx.x == 0) {
            if (loss) loss[r] = 0;
            stats[2 * int64_t(r)] = 0;
            stats[2 * int64_t(r) + 1] = 0;
        }
        return;
    }
    const T *row = z + zm(r);
    A best = -INFINITY;
    for (int64_t c = threadIdx.x; c < vocab; c += kThreads) best = MaxF()(best, to_acc<A>(row[c]));
    best = block_fold(MaxF(), best, buf);
    __syncthreads();
    A sum = 0;
    for (int64_t c = threadIdx.x; c < vocab; c += kThreads) {
        const A v = to_acc<A>(row[c]);
        sum += v == -INFINITY ? A(0) : exp_((v - best) * inv_temp);
    }
    sum = block_fold(SumF(), sum, buf);
    __syncthreads();
    const A log_sum = log_(sum);
    A s = 0;
    for (int i = threadIdx.x; i < k; i += kThreads) {
        if (t.at[i] < 0 || t.p[i] == 0) continue;
        const A v = to_acc<A>(row[t.at[i]]);
        s += t.p[i] * (t.logp[i] - (v == -INFINITY ? A(-INFINITY) : (v - best) * inv_temp - log_sum));
    }
    s = block_fold(SumF(), s, buf);
    if (threadIdx.x == 0) {
        if (loss) loss[r] = temp * temp * s;
        stats[2 * int64_t(r)] = best;
        stats[2 * int64_t(r) + 1] = log_sum;
    }
}

template <class T, class I>
__global__ void __launch_bounds__(kThreads) distillation_grad_kernel(const acc_t<T> *dloss, int64_t dstep,
                                                                     const T *z, RowMap zm, const acc_t<T> *top,
                                                                     const I *index, int k, int64_t vocab, acc_t<T> temp,
                                                                     acc_t<T> inv_temp, const acc_t<T> *stats, T *dz, RowMap dm)
{
    using A = acc_t<T>;
    __shared__ Teacher<A> t;
    __shared__ A buf[kThreads / 32];
    const uint32_t r = blockIdx.x;
    T *out = dz + dm(r);
    if (!load_teacher(t, top + int64_t(r) * k, index + int64_t(r) * k, k, vocab, inv_temp, buf)) {
        for (int64_t c = threadIdx.x; c < vocab; c += kThreads) out[c] = from_acc<T>(A(0));
        return;
    }
    const T *row = z + zm(r);
    const A best = stats[2 * int64_t(r)], log_sum = stats[2 * int64_t(r) + 1];
    const A g = dloss[r * dstep] * temp;
    // the first entry of each column takes all the teacher's weight on it
    for (int i = threadIdx.x; i < k; i += kThreads) {
        if (t.at[i] < 0) continue;
        A w = 0;
        bool first = true;
        for (int j = 0; j < k; ++j) {
            if (t.at[j] != t.at[i]) continue;
            first = first && j >= i;
            w += t.p[j];
        }
        if (!first) continue;
        const A v = to_acc<A>(row[t.at[i]]);
        const A q = v == -INFINITY ? A(0) : exp_((v - best) * inv_temp - log_sum);
        t.logp[i] = g * (q - w);
    }
    __syncthreads();
    for (int64_t c = threadIdx.x; c < vocab; c += kThreads) {
        const A v = to_acc<A>(row[c]);
        const A q = v == -INFINITY ? A(0) : exp_((v - best) * inv_temp - log_sum);
        out[c] = from_acc<T>(g * q);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < k; i += kThreads) {
        if (t.at[i] < 0) continue;
        bool first = true;
        for (int j = 0; j < i; ++j) first = first && t.at[j] != t.at[i];
        if (first) out[t.at[i]] = from_acc<T>(t.logp[i]);
    }
}

// --------------------------------------------------------------------------------------- launchers
struct DistilArgs {
    const dpb_array *z, *top, *index, *dloss, *stats, *loss, *dz;
    RowMap zm, dm;
    int64_t rows, vocab, k;
    double temp;
};

template <class T, class I> static int run_loss(const DistilArgs &a, acc_t<T> *stats, cudaStream_t s)
{
    using A = acc_t<T>;
    distillation_loss_kernel<T, I><<<static_cast<unsigned>(a.rows), kThreads, 0, s>>>(
        static_cast<const T *>(a.z->data), a.zm, static_cast<const A *>(a.top->data), static_cast<const I *>(a.index->data),
        static_cast<int>(a.k), a.vocab, A(a.temp), A(1.0 / a.temp), a.loss ? static_cast<A *>(a.loss->data) : nullptr, stats);
    note_kernel("distillation_loss");
    return check_launch("distillation_loss");
}

template <class T, class I> static int run_grad(const DistilArgs &a, const acc_t<T> *stats, cudaStream_t s)
{
    using A = acc_t<T>;
    distillation_grad_kernel<T, I><<<static_cast<unsigned>(a.rows), kThreads, 0, s>>>(
        static_cast<const A *>(a.dloss->data), a.dloss->nd == 0 ? 0 : 1, static_cast<const T *>(a.z->data), a.zm,
        static_cast<const A *>(a.top->data), static_cast<const I *>(a.index->data), static_cast<int>(a.k), a.vocab,
        A(a.temp), A(1.0 / a.temp), stats, static_cast<T *>(a.dz->data), a.dm);
    note_kernel("distillation_grad");
    return check_launch("distillation_grad");
}

template <class T, class I> static int run(const DistilArgs &a, cudaStream_t s)
{
    using A = acc_t<T>;
    if (a.stats && a.dz) return run_grad<T, I>(a, static_cast<const A *>(a.stats->data), s);
    if (a.stats) return run_loss<T, I>(a, static_cast<A *>(a.stats->data), s);
    void *work = nullptr;
    DPB_TRY(dpb_malloc(static_cast<size_t>(2 * a.rows) * sizeof(A), s, &work));
    int st = run_loss<T, I>(a, static_cast<A *>(work), s);
    if (st == DPB_OK && a.dz) st = run_grad<T, I>(a, static_cast<const A *>(work), s);
    dpb_free(work, s);
    return st;
}

static int run_typed(const DistilArgs &a, cudaStream_t s)
{
    const bool narrow = a.index->typenum == DPB_INT32;
    switch (a.z->typenum) {
    case DPB_HALF: return narrow ? run<half_t, int32_t>(a, s) : run<half_t, int64_t>(a, s);
    case DPB_FLOAT: return narrow ? run<float, int32_t>(a, s) : run<float, int64_t>(a, s);
    default: return narrow ? run<double, int32_t>(a, s) : run<double, int64_t>(a, s);
    }
}

// Checks shared by the three entry points; the row maps are filled when there are rows.
static int check_args(DistilArgs &a)
{
    const dpb_array &z = *a.z;
    DPB_TRY(check_float_type(z, "logits"));
    if (z.nd < 1) return set_error(DPB_ERR_VALUE, "logits: an array of at least one dimension is needed");
    const int lead = z.nd - 1, at = acc_typenum(z.typenum);
    a.rows = count_rows(z);
    a.vocab = z.shape[lead];
    if (a.vocab == 0) return set_error(DPB_ERR_VALUE, "the loss cannot be taken over zero-size axes");
    if (a.rows > kMaxRows) return set_error(DPB_ERR_VALUE, "more than 2^31 - 1 rows are not supported");
    DPB_TRY(check_operand(a.top, "teacher_logits"));
    DPB_TRY(check_operand(a.index, "teacher_index"));
    if (a.top->nd < 1) return set_error(DPB_ERR_VALUE, "teacher_logits: an array of at least one dimension is needed");
    a.k = a.top->shape[a.top->nd - 1];
    if (a.k > kMaxTop) return set_error(DPB_ERR_VALUE, "at most %d teacher entries a row are supported, got %lld", kMaxTop, static_cast<long long>(a.k));
    DPB_TRY(check_type(*a.top, at, "teacher_logits"));
    DPB_TRY(check_shape(*a.top, z.shape, lead, a.k, "teacher_logits"));
    DPB_TRY(check_c_contiguous(*a.top, "teacher_logits"));
    if (a.index->typenum != DPB_INT32 && a.index->typenum != DPB_INT64)
        return set_error(DPB_ERR_TYPE, "teacher_index: int32 or int64 is needed, got %s", type_name(a.index->typenum));
    DPB_TRY(check_shape(*a.index, z.shape, lead, a.k, "teacher_index"));
    DPB_TRY(check_c_contiguous(*a.index, "teacher_index"));
    // T^2 and 1/T have to be ordinary numbers of the type that the loss is computed in
    const double t = a.temp;
    bool fits = t > 0 && std::isfinite(t);
    if (at == DPB_FLOAT) {
        const float f = static_cast<float>(t), inv = static_cast<float>(1.0 / t);
        fits = fits && std::isnormal(f * f) && std::isnormal(inv);
    }
    else fits = fits && std::isnormal(t * t) && std::isnormal(1.0 / t);
    if (!fits) return set_error(DPB_ERR_VALUE, "temperature must be a positive number within the range of the computation");
    for (const dpb_array *x : {a.top, a.index}) DPB_TRY(check_same_device(z, *x));
    if (a.dloss) {
        DPB_TRY(check_operand(a.dloss, "dloss"));
        DPB_TRY(check_same_device(z, *a.dloss));
        DPB_TRY(check_type(*a.dloss, at, "dloss"));
        if (a.dloss->nd != 0) DPB_TRY(check_shape(*a.dloss, z.shape, lead, -1, "dloss"));
        DPB_TRY(check_c_contiguous(*a.dloss, "dloss"));
    }
    if (a.stats) {
        DPB_TRY(check_operand(a.stats, "stats"));
        DPB_TRY(check_same_device(z, *a.stats));
        DPB_TRY(check_type(*a.stats, at, "stats"));
        DPB_TRY(check_shape(*a.stats, z.shape, lead, 2, "stats"));
        DPB_TRY(check_c_contiguous(*a.stats, "stats"));
    }
    if (a.loss) {
        DPB_TRY(check_operand(a.loss, "loss"));
        DPB_TRY(check_same_device(z, *a.loss));
        DPB_TRY(check_type(*a.loss, at, "loss"));
        DPB_TRY(check_shape(*a.loss, z.shape, lead, -1, "loss"));
        DPB_TRY(check_c_contiguous(*a.loss, "loss"));
        DPB_TRY(check_output(*a.loss, "loss"));
    }
    if (a.dz) {
        DPB_TRY(check_operand(a.dz, "dlogits"));
        DPB_TRY(check_same_device(z, *a.dz));
        DPB_TRY(check_type(*a.dz, z.typenum, "dlogits"));
        DPB_TRY(check_shape(*a.dz, z.shape, z.nd, -1, "dlogits"));
        DPB_TRY(check_output(*a.dz, "dlogits"));
        DPB_TRY(check_no_overlap(z, *a.dz, true));
    }
    if (a.rows > 0) {
        DPB_TRY(check_row_map(z, a.zm, "logits"));
        if (a.dz) DPB_TRY(check_row_map(*a.dz, a.dm, "dlogits"));
    }
    return DPB_OK;
}

}  // namespace dpb

using namespace dpb;

extern "C" {

int dpb_distillation_loss(const dpb_array *logits, const dpb_array *teacher_logits, const dpb_array *teacher_index,
                          double temperature, const dpb_array *loss, const dpb_array *stats, void *stream)
{
    DPB_TRY(check_operand(logits, "logits"));
    DPB_TRY(check_operand(loss, "loss"));
    DistilArgs a = {};
    a.z = logits, a.top = teacher_logits, a.index = teacher_index, a.temp = temperature, a.loss = loss, a.stats = stats;
    DPB_TRY(check_args(a));
    if (stats) DPB_TRY(check_output(*stats, "stats"));
    DPB_TRY(check_no_overlaps({logits, teacher_logits, teacher_index}, {loss, stats}));
    return a.rows == 0 ? DPB_OK : run_typed(a, static_cast<cudaStream_t>(stream));
}

int dpb_distillation_loss_backward(const dpb_array *dloss, const dpb_array *logits, const dpb_array *teacher_logits,
                                   const dpb_array *teacher_index, const dpb_array *stats, double temperature,
                                   const dpb_array *dlogits, void *stream)
{
    DPB_TRY(check_operand(logits, "logits"));
    DPB_TRY(check_operand(dloss, "dloss"));
    DPB_TRY(check_operand(stats, "stats"));
    DPB_TRY(check_operand(dlogits, "dlogits"));
    DistilArgs a = {};
    a.z = logits, a.top = teacher_logits, a.index = teacher_index, a.temp = temperature, a.dloss = dloss, a.stats = stats,
    a.dz = dlogits;
    DPB_TRY(check_args(a));
    DPB_TRY(check_no_overlaps({teacher_logits, teacher_index, dloss, stats}, {dlogits}));
    return a.rows == 0 ? DPB_OK : run_typed(a, static_cast<cudaStream_t>(stream));
}

int dpb_distillation_loss_and_grad(const dpb_array *logits, const dpb_array *teacher_logits, const dpb_array *teacher_index,
                                   const dpb_array *dloss, double temperature, const dpb_array *loss,
                                   const dpb_array *dlogits, void *stream)
{
    DPB_TRY(check_operand(logits, "logits"));
    DPB_TRY(check_operand(dloss, "dloss"));
    DPB_TRY(check_operand(loss, "loss"));
    DPB_TRY(check_operand(dlogits, "dlogits"));
    DistilArgs a = {};
    a.z = logits, a.top = teacher_logits, a.index = teacher_index, a.temp = temperature, a.dloss = dloss, a.loss = loss,
    a.dz = dlogits;
    DPB_TRY(check_args(a));
    DPB_TRY(check_no_overlaps({logits, teacher_logits, teacher_index, dloss}, {loss}));
    DPB_TRY(check_no_overlaps({teacher_logits, teacher_index, dloss}, {loss, dlogits}));
    return a.rows == 0 ? DPB_OK : run_typed(a, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
