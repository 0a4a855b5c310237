// Distillation loss from a teacher's top logits, and its gradient.
//
// Row r has V student logits z and K teacher logits t at columns j.  An entry counts when 0 <= j < V
// and t > -inf.  With a temperature T,
//   p = softmax(t / T) over the entries that count,  q = softmax(z / T),
//   loss = T^2 sum_k p_k (log p_k - log q_{j_k}),    dz = dloss T (q - sum_{k: j_k = .} p_k).
// A row without entries (padding, a prompt) has loss 0 and gradient 0, whatever its logits.
// Where q is 0 (z = -inf, or every z of the row) and p is not, the loss is +inf; q counts as 0 in dz.
//
// log q = (z - max z) / T - log sum exp((z - max z) / T): the differences are taken before the division, and the
// terms of the loss are T (log p - log q), so that logits of the type's lowest value do not overflow.  The two
// statistics (max z, log of the sum) are kept apart for the backward pass: their sum would lose log2 |max z| bits.
// All of it is float (double for float64 logits); each gradient is rounded once.
#include "row_ops.cuh"

namespace dpb {

constexpr int kMaxTop = 1024;   // teacher entries a row may have

DPB_D float max_nan(float a, float b)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
DPB_D double max_nan(double a, double b) { return MaxF()(a, b); }
struct MaxNanF {
    template <class A> DPB_D A operator()(A a, A b) const { return max_nan(a, b); }
};
// 2^a: within 2^-22 for float (the instruction; FTZ: results below 2^-126 are zero).
template <bool FTZ> DPB_D float exp2_(float a)
{
    float r;
    if constexpr (FTZ) asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(a));
    else asm("ex2.approx.f32 %0, %1;" : "=f"(r) : "f"(a));
    return r;
}
template <bool FTZ> DPB_D double exp2_(double a) { return exp2(a); }
constexpr double kLog2E = 1.4426950408889634074;

// Exponentials of a row's values below its largest one, T given as k = log2(e) / T.
//
// 2^((v - top) k), the difference taken first, so that values of the type's lowest number do not overflow.  FUSED,
// for float16: 2^(v k - c) with c = top k rounded, which is one operation a value; what c is off by (rest) is exact
// and corrects the sum once.  `finite`: what a row whose values are all -inf is reduced by.
template <class T, bool FUSED> struct Exponent {
    using A = acc_t<T>;
    static constexpr bool fused = FUSED;
    A k, base;
    static DPB_D A finite(A t) { return t == -INFINITY ? A(0) : t; }
    DPB_D Exponent(A top, A k_) : k(k_), base(fused ? -(finite(top) * k_) : -finite(top)) {}
    template <bool FTZ> DPB_D A exp(A v) const
    {
        return exp2_<FTZ>(fused ? fma_(v, k, base) : (v + base) * k);
    }
    template <bool FTZ, int N> DPB_D void exp(Values<A, N> &v) const
    {
        Values<A, N> e;
        if constexpr (fused) {
            e.fill(base);
            e.fma_add(v, k);
        }
        else {
            e = v;
            e.add(base);
            e.mul(k);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) v.set(i, exp2_<FTZ>(e.get(i)));
    }
    // log2 of the factor between the sum of these exponentials and that of exp((v - top) / T)
    DPB_D A rest(A top) const { return fused ? fma_(finite(top), k, base) : A(0); }
};

// The largest of some values and the sum of their exponentials.
template <class T, bool FUSED> struct alignas(2 * sizeof(acc_t<T>)) SoftSum {
    using A = acc_t<T>;
    using Exp = Exponent<T, FUSED>;
    A top, sum;
    DPB_D void raise(A to, A k)   // to >= top
    {
        if constexpr (FUSED) {
            const A factor = exp2_<true>(Exp(to, k).base - Exp(top, k).base);
            sum = top == -INFINITY ? A(0) : sum * factor;
        }
        else sum *= exp2_<true>((top - Exp::finite(to)) * k);
        top = to;
    }
    DPB_D SoftSum over_warp(A k) const
    {
        SoftSum s = *this;
        s.raise(warp_fold(MaxNanF(), top), k);
        s.sum = warp_fold(SumF(), s.sum);
        return s;
    }
    DPB_D A log_sum(A k) const   // log sum exp((v - top) / T)
    {
        return log_(sum) - Exp(top, k).rest(top) * A(0.69314718055994530942);
    }
};

// Largest of the values of an access, NaN if there is one.
template <class T, int N> DPB_D acc_t<T> largest(const vec_t<T, N> &raw)
{
    if constexpr (is_half_v<T>) {
        const __half2 *h = reinterpret_cast<const __half2 *>(raw.v);
        __half2 m = h[0];
#pragma unroll
        for (int i = 1; i < N / 2; ++i) m = __hmax2_nan(m, h[i]);
        return __half2float(__hmax_nan(__low2half(m), __high2half(m)));
    }
    else {
        acc_t<T> m = raw.v[0];
#pragma unroll
        for (int i = 1; i < N; ++i) m = max_nan(m, raw.v[i]);
        return m;
    }
}

// A row's teacher as a block keeps it: probability, its logarithm and column (-1: does not count) of each entry.
template <class A> struct Teacher {
    A *p, *logp;
    int *at;
    static DPB_HD size_t bytes(int k) { return size_t(k) * (2 * sizeof(A) + sizeof(int)) + 16; }
    DPB_D Teacher(void *shared, int k) : p(static_cast<A *>(shared)), logp(p + k), at(reinterpret_cast<int *>(logp + k)) {}
    // The block reads the entries (thread t every blockDim.x-th from t on); false for all when none counts.
    template <class I> DPB_D bool read(const A *top, const I *index, int k, int vocab) const
    {
        bool any = false;
        for (int i = threadIdx.x; i < k; i += blockDim.x) {
            const A v = top[i];
            const int64_t j = static_cast<int64_t>(index[i]);
            const bool counts = j >= 0 && j < vocab && !(v == -INFINITY);
            at[i] = counts ? static_cast<int>(j) : -1;
            logp[i] = v;
            any = any || counts;
        }
        return __syncthreads_or(any);
    }
    // One warp turns them into probabilities.
    DPB_D void normalize(int k, A inv_temp) const
    {
        const int lane = threadIdx.x & 31;
        A best = -INFINITY, sum = 0;
        for (int i = lane; i < k; i += 32)
            if (at[i] >= 0) best = max_nan(best, logp[i]);
        best = warp_fold(MaxNanF(), best);
        for (int i = lane; i < k; i += 32) {
            const A e = at[i] >= 0 ? exp_((logp[i] - best) * inv_temp) : A(0);
            p[i] = e;
            sum += e;
        }
        sum = warp_fold(SumF(), sum);
        const A log_sum = log_(sum);
        for (int i = lane; i < k; i += 32) {
            p[i] = p[i] / sum;
            logp[i] = at[i] >= 0 ? (logp[i] - best) * inv_temp - log_sum : A(0);
        }
    }
    // All the weight on the column of entry i; false when an earlier entry has the same column.  K comparisons an entry:
    // little up to some hundred entries, the greater part of the time at 1024 (4096 x 128000 float16, gradient alone: 330 us
    // with 64 entries, 383 with 256, 3091 with 1024; with the loss 393, 621 and 5960).
    DPB_D bool first_of_column(int i, int k, A &weight) const
    {
        bool first = true;
        weight = 0;
        for (int j = 0; j < k; ++j) {
            if (at[j] != at[i]) continue;
            first = first && j >= i;
            weight += p[j];
        }
        return first;
    }
};

// How rows are shared out: 2^bits blocks (ranks) a row, `each` accesses a rank at most.
struct Shares {
    int bits, each;
    DPB_D uint32_t row() const { return blockIdx.x >> bits; }
    DPB_D int rank() const { return blockIdx.x & ((1 << bits) - 1); }
};

// A row of V logits as whole accesses of 16 bytes behind `head` single elements, `tail` elements behind them; a rank has
// `mine` accesses, the first of which starts at column `first`.
template <class T> struct RowSplit {
    static constexpr int VEC = vec_width<T>();
    int head, tail, first, mine;
    DPB_D RowSplit(const T *row, int vocab, const Shares &sh)
    {
        const int off = misalignment(row), rank = sh.rank();
        head = min(vocab, off ? VEC - off : 0);
        const int all = (vocab - head) / VEC, begin = min(all, sh.each * rank);
        tail = vocab - head - all * VEC;
        mine = min(all, begin + sh.each) - begin;
        first = head + begin * VEC;
        if (rank > 0) head = 0;
        if (rank < (1 << sh.bits) - 1) tail = 0;
    }
    // The thread's single element (head or tail), as a column; -1 without one.
    DPB_D int single(int vocab) const
    {
        const int t = threadIdx.x;
        return t < head ? t : t < head + tail ? vocab - tail + (t - head) : -1;
    }
};

// The gradient of a row's columns, dloss T (q - weight): q is an exponential times `scale` (0 in a row whose logits
// are all -inf).
template <class T, bool FUSED> struct RowGradient {
    using A = acc_t<T>;
    static constexpr bool ftz = is_half_v<T>;   // (float16 has no numbers as small as those that are flushed)
    Exponent<T, FUSED> ex;
    A scale, g;
    DPB_D RowGradient(const SoftSum<T, FUSED> &s, A k, A g_) : ex(s.top, k), scale(s.sum == 0 ? A(0) : g_ / s.sum), g(g_) {}
    DPB_D RowGradient(A top, A log_sum, A k, A g_)   // from kept statistics
        : ex(top, k), scale(log_sum == -INFINITY ? A(0) : g_ * exp_(-log_sum) * exp2_<false>(-ex.rest(top))), g(g_)
    {
    }
    DPB_D A at(A v, A weight) const { return ex.template exp<ftz>(v) * scale - g * weight; }
    template <int N> DPB_D void apply(Values<A, N> &v) const
    {
        ex.template exp<ftz>(v);
        v.mul(scale);
    }
};

// ------------------------------------------------------------------------------------------- a row's parts
constexpr int kThreads = 256;   // of a block, at most
constexpr int kInFlight = 4;    // accesses of a thread
constexpr int kMaxRanks = 8;    // blocks of a cluster

// What a block of either kernel below knows of its part of a row, and its work on it.
template <class T, class I> struct RowPart {
    using A = acc_t<T>;
    static constexpr int VEC = vec_width<T>();
    using V = vec_t<T, VEC>;
    const T *row;
    RowSplit<T> split;
    Teacher<A> teacher;
    A *at_teacher;   // the student's logits at the teacher's columns
    int single, k, vocab;

    static DPB_HD size_t shared_bytes(int k) { return (Teacher<A>::bytes(k) + 15) / 16 * 16 + size_t(k) * sizeof(A); }
    DPB_D RowPart(const T *row_, int vocab_, int k_, const Shares &share, char *shared)
        : row(row_), split(row_, vocab_, share), teacher(shared, k_),
          at_teacher(reinterpret_cast<A *>(shared + (Teacher<A>::bytes(k_) + 15) / 16 * 16)), single(split.single(vocab_)), k(k_), vocab(vocab_)
    {
    }
    DPB_D bool owns(int c) const
    {
        return (c >= split.first && c < split.first + split.mine * VEC) || (c >= 0 && c < split.head) || c >= vocab - split.tail;
    }
    // The student's logit at the column of an entry that this thread has read (`all`, or this part's).
    DPB_D T student(int i, bool all) const
    {
        const int c = i < k ? teacher.at[i] : -1;
        return c >= 0 && (all || owns(c)) ? row[c] : from_acc<T>(A(0));
    }
    DPB_D const V *from() const { return reinterpret_cast<const V *>(row + split.first); }
    // Stores that are not read again here: they leave the cache first.
    DPB_D void put(T *out, int i, const V &v, bool aligned) const
    {
        T *o = out + split.first + i * VEC;
        if (aligned) __stcs(reinterpret_cast<int4 *>(o), reinterpret_cast<const int4 &>(v));
        else
#pragma unroll
            for (int j = 0; j < VEC; ++j) o[j] = v.v[j];
    }
    DPB_D bool aligned(const T *out) const { return split.mine > 0 && misalignment(out + split.first) == 0; }
    DPB_D void zeros(T *out) const
    {
        const bool whole = aligned(out);
        V z;
#pragma unroll
        for (int j = 0; j < VEC; ++j) z.v[j] = from_acc<T>(A(0));
        for (int i = threadIdx.x; i < split.mine; i += blockDim.x) put(out, i, z, whole);
        if (single >= 0) out[single] = z.v[0];
    }
    // Whether the part starts on a cache line.
    DPB_D bool on_lines() const { return reinterpret_cast<uintptr_t>(from()) % 128 == 0; }
    // LAST: lines leave the cache as they are read (16384 x 32000 float16: 358 us against 370), but not where two warps
    // share a line, which the second would miss (16384 x 50257 float16: 671 us against 636).
    template <bool LAST, bool FUSED> DPB_D void dense_gradient(T *out, const RowGradient<T, FUSED> &grad) const
    {
        const bool whole = aligned(out);
        const int threads = blockDim.x;
        const V *p = from();
        for (int i0 = threadIdx.x; i0 < split.mine; i0 += kInFlight * threads) {
            V raw[kInFlight];
#pragma unroll
            for (int f = 0; f < kInFlight; ++f)
                if (i0 + f * threads < split.mine) {
                    if constexpr (LAST) reinterpret_cast<int4 &>(raw[f]) = __ldcs(reinterpret_cast<const int4 *>(p + i0 + f * threads));
                    else raw[f] = p[i0 + f * threads];
                }
#pragma unroll
            for (int f = 0; f < kInFlight; ++f) {
                if (i0 + f * threads >= split.mine) break;
                Values<A, VEC> v;
                unpack<A, VEC, T>(raw[f], v);
                grad.apply(v);
                put(out, i0 + f * threads, repack<T, VEC, A>(v), whole);
            }
        }
        if (single >= 0) out[single] = from_acc<T>(grad.at(to_acc<A>(row[single]), A(0)));
    }
    // The teacher's columns of this part once more, with its weight taken off (after a barrier).
    template <bool FUSED> DPB_D void teacher_gradient(T *out, const RowGradient<T, FUSED> &grad) const
    {
        for (int i = threadIdx.x; i < k; i += blockDim.x) {
            const int c = teacher.at[i];
            if (c < 0 || !owns(c)) continue;
            A weight;
            if (teacher.first_of_column(i, k, weight)) out[c] = from_acc<T>(grad.at(at_teacher[i], weight));
        }
    }
};

// --------------------------------------------------------------------------------- loss, and loss and gradient
// A cluster of 1 to 8 blocks takes a row: every block streams its part (largest value and sum of exponentials, both per
// thread), the blocks exchange their sums through distributed shared memory, and (GRAD) read their parts again,
// from the second-level cache, for the gradient: with parts of 64 KiB the clusters that run at a time hold 30 to 60 MB,
// which the cache keeps, and the logits cross the memory once.  That holds for rows of up to 512 KiB.  The parts of longer
// rows grow, and the second reading misses: 1024 x 131072 float32 reads 1.04 times the logits (197 us, 0.83 of the copy
// rate), 1024 x 150001 1.20 times (242 us, 0.78), 512 x 300000 1.98 times (307 us, 0.61).  float64 is bound by its
// exponentials (512 x 150001: loss 192 us, gradient 252 us, both 428 us).  4096 x 128000 float16 takes 400 us (0.80); the
// parts kept in shared memory instead, by copies that run ahead, 487 us, because few threads fit beside them; clusters
// that stay and fetch the next row's teacher ahead, 766 us, because they read and write in step.  What a block waits for
// beside its part counts as much as the bytes: the first logits are fetched with the teacher's entries, the student's
// logits at their columns arrive while the part is streamed, and one warp forms the probabilities and the loss while the
// others go on (418 us with these one after the other; 1024 x 150001 float32 timed one by one: 288, now 264).
//
// Two exponentials an element: at float16 and the copy rate that is 3.3e12 a second, three quarters of what the
// special function units give; the rest of the arithmetic is done in pairs to stay out of their way.
template <class T, class I, bool GRAD, bool FUSED>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 8 ? 4 : 6)
    distillation_row_kernel(const T *z, RowMap zm, const acc_t<T> *top, const I *index, int k, int vocab, acc_t<T> temp,
                            acc_t<T> inv_temp, acc_t<T> exp_scale, acc_t<T> *loss, acc_t<T> *stats, const acc_t<T> *dloss,
                            int64_t dstep, T *dz, RowMap dm, Shares share)
{
    using A = acc_t<T>;
    using Part = RowPart<T, I>;
    using Sum = SoftSum<T, FUSED>;
    using V = typename Part::V;
    constexpr int VEC = Part::VEC;
    extern __shared__ __align__(16) char shared_bytes[];
    __shared__ Sum warp_sums[kThreads / 32], rank_sums[kMaxRanks];
    cudaGridDependencySynchronize();
    const uint32_t r = share.row();
    const int rank = share.rank(), ranks = 1 << share.bits, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, threads = blockDim.x;
    const Part part(z + zm(r), vocab, k, share, shared_bytes);
    T *out = GRAD ? dz + dm(r) : nullptr;
    const V *from = part.from();
    V raw[kInFlight], low;
#pragma unroll
    for (int j = 0; j < VEC; ++j) low.v[j] = from_acc<T>(A(-INFINITY));
    const auto load = [&](int i0) {
#pragma unroll
        for (int f = 0; f < kInFlight; ++f) raw[f] = i0 + f * threads < part.split.mine ? from[i0 + f * threads] : low;
    };
    load(threadIdx.x);   // while the teacher's entries are on their way
    if (!part.teacher.read(top + int64_t(r) * k, index + int64_t(r) * k, k, vocab)) {   // every block of the cluster
        if (rank == 0 && threadIdx.x == 0) {
            if (loss) loss[r] = 0;
            if (stats) stats[2 * int64_t(r)] = stats[2 * int64_t(r) + 1] = 0;
        }
        if constexpr (GRAD) part.zeros(out);
        return;
    }
    // (waited for before the first write into another block's memory: that block has to have begun)
    if (ranks > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    const T student = part.student(threadIdx.x, rank == 0);
    const A alone = part.single >= 0 ? to_acc<A>(part.row[part.single]) : A(-INFINITY);
    Sum s = {alone, part.single >= 0 ? Exponent<T, FUSED>(alone, exp_scale).template exp<true>(alone) : A(0)};
    for (int i0 = threadIdx.x; i0 < part.split.mine; i0 += kInFlight * threads) {
        A best = largest<T, VEC>(raw[0]);
#pragma unroll
        for (int f = 1; f < kInFlight; ++f) best = max_nan(best, largest<T, VEC>(raw[f]));
        s.raise(max_nan(s.top, best), exp_scale);
        const Exponent<T, FUSED> ex(s.top, exp_scale);
        auto sum = Values<A, VEC>::all(0);
#pragma unroll
        for (int f = 0; f < kInFlight; ++f) {
            Values<A, VEC> v;
            unpack<A, VEC, T>(raw[f], v);
            ex.template exp<true>(v);
            v.sum_into(sum);
        }
        s.sum += Values<A, VEC>::join(sum);
        load(i0 + kInFlight * threads);
    }
    // before any block writes over the logits
    if (threadIdx.x < k) part.at_teacher[threadIdx.x] = to_acc<A>(student);
    for (int i = threadIdx.x + threads; i < k; i += threads) part.at_teacher[i] = to_acc<A>(part.student(i, rank == 0));
    // lanes, warps and ranks, each in a fixed order
    s = s.over_warp(exp_scale);
    if (lane == 0) warp_sums[warp] = s;
    __syncthreads();
    s = lane < threads / 32 ? warp_sums[lane] : Sum{-INFINITY, 0};
    s = s.over_warp(exp_scale);
    if (ranks > 1) {
        asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
        // every rank writes its sum to every rank; the barrier of the cluster makes them visible (and follows the
        // reads of the student's logits)
        if (threadIdx.x < ranks) {
            const uint32_t local = static_cast<uint32_t>(__cvta_generic_to_shared(&rank_sums[rank]));
            uint32_t remote;
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(threadIdx.x));
            if constexpr (sizeof(A) == 4)
                asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(remote), "f"(s.top), "f"(s.sum) : "memory");
            else
                asm volatile("st.shared::cluster.v2.f64 [%0], {%1, %2};" ::"r"(remote), "d"(s.top), "d"(s.sum) : "memory");
        }
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        s = lane < ranks ? rank_sums[lane] : Sum{-INFINITY, 0};
        s = s.over_warp(exp_scale);
    }
    if (warp == 0) {   // the other warps go on
        part.teacher.normalize(k, inv_temp);
        const A log_sum = s.log_sum(exp_scale);
        A total = 0;
        if (rank == 0) {
            for (int i = lane; i < k; i += 32) {
                if (part.teacher.at[i] < 0 || part.teacher.p[i] == 0) continue;
                // T (log p - log q): the depth of the logit is not divided by T, which below 1 would take that of a
                // logit of the type's lowest value out of range
                const A v = part.at_teacher[i];
                total += part.teacher.p[i] *
                         (v == -INFINITY ? A(INFINITY) : temp * (part.teacher.logp[i] + log_sum) + (s.top - v));
            }
            total = warp_fold(SumF(), total);
        }
        if (rank == 0 && lane == 0) {
            if (loss) loss[r] = temp * total;
            if (stats) {
                stats[2 * int64_t(r)] = s.top;
                stats[2 * int64_t(r) + 1] = log_sum;
            }
        }
    }
    if constexpr (GRAD) {
        const RowGradient<T, FUSED> grad(s, exp_scale, dloss[r * dstep] * temp);
        if (part.on_lines()) part.template dense_gradient<true>(out, grad);
        else part.template dense_gradient<false>(out, grad);
        __syncthreads();
        part.teacher_gradient(out, grad);
    }
}

// ------------------------------------------------------------------------------------------ gradient alone
// From kept statistics: the same parts, without exchange.
template <class T, class I, bool FUSED>
__global__ void __launch_bounds__(kThreads)
    distillation_grad_kernel(const acc_t<T> *dloss, int64_t dstep, const T *z, RowMap zm, const acc_t<T> *top, const I *index, int k,
                             int vocab, acc_t<T> temp, acc_t<T> inv_temp, acc_t<T> exp_scale, const acc_t<T> *stats, T *dz,
                             RowMap dm, Shares share)
{
    using A = acc_t<T>;
    extern __shared__ __align__(16) char shared_bytes[];
    cudaGridDependencySynchronize();
    const uint32_t r = share.row();
    const RowPart<T, I> part(z + zm(r), vocab, k, share, shared_bytes);
    T *out = dz + dm(r);
    if (!part.teacher.read(top + int64_t(r) * k, index + int64_t(r) * k, k, vocab)) return part.zeros(out);
    for (int i = threadIdx.x; i < k; i += blockDim.x) part.at_teacher[i] = to_acc<A>(part.student(i, false));
    __syncthreads();
    const RowGradient<T, FUSED> grad(stats[2 * int64_t(r)], stats[2 * int64_t(r) + 1], exp_scale, dloss[r * dstep] * temp);
    part.template dense_gradient<false>(out, grad);
    if (threadIdx.x < 32) part.teacher.normalize(k, inv_temp);
    __syncthreads();
    part.teacher_gradient(out, grad);
}

// --------------------------------------------------------------------------------------- launchers
struct DistilArgs {
    const dpb_array *z, *top, *index, *dloss, *stats, *loss, *dz;
    RowMap zm, dm;
    int64_t rows, vocab, k;
    double temp;
};

// Blocks that share a row: parts of `part` bytes at most, at most 2^most of them; few rows are split further, down to 8
// KiB.
static int share_row(const DistilArgs &a, int item, int64_t part, int most, Shares &share)
{
    const int64_t bytes = a.vocab * item, vec = 16 / item;
    share.bits = 0;
    while (share.bits < most && (bytes >> share.bits) > part) ++share.bits;
    while (share.bits < most && (a.rows << share.bits) < 4 * device_props().sm_count && (bytes >> share.bits) >= 16 * 1024) ++share.bits;
    if ((a.rows << share.bits) > INT32_MAX) return set_error(DPB_ERR_VALUE, "too many rows of this length");
    share.each = static_cast<int>(ceil_div(a.vocab / vec, int64_t(1) << share.bits));
    return DPB_OK;
}

// Threads of a block: up to two rounds of kInFlight accesses each before the block grows (short rows gain from more
// blocks on an SM: 8192 x 5000 float16 takes 80 us with 256 threads, 49 with 128), at least two warps.
static unsigned share_threads(const Shares &share)
{
    unsigned threads = 64;
    while (threads < unsigned(kThreads) && share.each > 2 * kInFlight * static_cast<int>(threads)) threads *= 2;
    return threads;
}

template <class T, class I, bool FUSED> static int run_grad(const DistilArgs &a, cudaStream_t s)
{
    using A = acc_t<T>;
    Shares share;
    // parts of 64 to 128 KiB: below that the teacher's entries, which every block reads, show (1024 x 150001 float32:
    // 221 us at 75 KiB, 266 us at 37 KiB)
    DPB_TRY(share_row(a, sizeof(T), 128 * 1024, 10, share));
    launch_shared<distillation_grad_kernel<T, I, FUSED>>(
        static_cast<unsigned>(a.rows << share.bits), share_threads(share), RowPart<T, I>::shared_bytes(int(a.k)), s,
        static_cast<const A *>(a.dloss->data), a.dloss->nd == 0 ? 0 : 1, static_cast<const T *>(a.z->data), a.zm,
        static_cast<const A *>(a.top->data), static_cast<const I *>(a.index->data), static_cast<int>(a.k),
        static_cast<int>(a.vocab), A(a.temp), A(1.0 / a.temp), A(kLog2E / a.temp), static_cast<const A *>(a.stats->data),
        static_cast<T *>(a.dz->data), a.dm, share);
    note_kernel("distillation_grad");
    return check_launch("distillation_grad");
}

template <class T, class I, bool GRAD, bool FUSED> static int run_rows(const DistilArgs &a, cudaStream_t s)
{
    using A = acc_t<T>;
    Shares share;
    // Loss: whole rows (4096 x 128000 float16: 181 us, 185 with halves, 212 with quarters; 8192 x 150001 float32: 715 us,
    // 900 with quarters).  Loss and gradient: what the clusters hold has to stay in the cache between the two readings
    // (4096 x 128000 float16: 400 us with quarters, 476 with halves).
    DPB_TRY(share_row(a, sizeof(T), GRAD ? 64 * 1024 : INT64_MAX, 3, share));
    launch_cluster<distillation_row_kernel<T, I, GRAD, FUSED>>(
        static_cast<unsigned>(a.rows << share.bits), 1u << share.bits, share_threads(share),
        RowPart<T, I>::shared_bytes(int(a.k)), s, static_cast<const T *>(a.z->data), a.zm,
        static_cast<const A *>(a.top->data), static_cast<const I *>(a.index->data), static_cast<int>(a.k),
        static_cast<int>(a.vocab), A(a.temp), A(1.0 / a.temp), A(kLog2E / a.temp),
        a.loss ? static_cast<A *>(a.loss->data) : nullptr, a.stats ? static_cast<A *>(a.stats->data) : nullptr,
        GRAD ? static_cast<const A *>(a.dloss->data) : nullptr, GRAD && a.dloss->nd > 0 ? 1 : 0,
        GRAD ? static_cast<T *>(a.dz->data) : nullptr, a.dm, share);
    note_kernel("distillation_row");
    return check_launch("distillation_row");
}

template <class T, class I, bool FUSED> static int run_as(const DistilArgs &a, cudaStream_t s)
{
    if (a.dz && !a.loss) return run_grad<T, I, FUSED>(a, s);
    return a.dz ? run_rows<T, I, true, FUSED>(a, s) : run_rows<T, I, false, FUSED>(a, s);
}

template <class T, class I> static int run(const DistilArgs &a, cudaStream_t s)
{
    if constexpr (is_half_v<T>) {
        // While the largest float16 divided by T (in powers of two) is below 2^24, its rounding is at most half a power
        // of two.  Colder, the factor that corrects it would leave the range of float.
        if (65504 * kLog2E / a.temp < 16777216) return run_as<T, I, true>(a, s);
    }
    return run_as<T, I, false>(a, s);
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
    if (a.rows > kMaxRows || a.vocab > kMaxRows)
        return set_error(DPB_ERR_VALUE, "more than 2^31 - 1 rows or columns are not supported");
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
