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

// The largest value and the sum of exp((v - largest) / T) of some values, T given as k = log2(e) / T.
template <class A> struct alignas(2 * sizeof(A)) SoftSum {
    A top, sum;
    // what v is reduced by: a finite number even where every value is -inf
    static DPB_D A finite(A t) { return t == -INFINITY ? A(0) : t; }
    DPB_D void raise(A to, A k)   // to >= top
    {
        sum *= exp2_<true>((top - finite(to)) * k);
        top = to;
    }
    DPB_D SoftSum over_warp(A k) const
    {
        SoftSum s = *this;
        s.raise(warp_fold(MaxNanF(), top), k);
        s.sum = warp_fold(SumF(), s.sum);
        return s;
    }
};

// A row's teacher as a block keeps it: probability, its logarithm and column (-1: does not count) of each entry.
template <class A> struct Teacher {
    A *p, *logp;
    int *at;
    static DPB_HD size_t bytes(int k) { return size_t(k) * (2 * sizeof(A) + sizeof(int)) + 16; }
    DPB_D Teacher(void *shared, int k) : p(static_cast<A *>(shared)), logp(p + k), at(reinterpret_cast<int *>(logp + k)) {}
    // One warp reads the entries; false when none counts.
    template <class I> DPB_D bool read(const A *top, const I *index, int k, int64_t vocab) const
    {
        bool any = false;
        for (int i = threadIdx.x & 31; i < k; i += 32) {
            const A v = top[i];
            const int64_t j = static_cast<int64_t>(index[i]);
            const bool counts = j >= 0 && j < vocab && !(v == -INFINITY);
            at[i] = counts ? static_cast<int>(j) : -1;
            logp[i] = v;
            any = any || counts;
        }
        return __any_sync(0xffffffffu, any);
    }
    // The same warp turns them into probabilities.
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
    // All the weight on the column of entry i; false when an earlier entry has the same column.
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

// A row of V logits as whole accesses of 16 bytes behind `head` single elements, `tail` elements behind them; a
// rank (of `ranks` blocks) has `mine` accesses from access `begin` on.
template <class T> struct RowSplit {
    static constexpr int VEC = vec_width<T>();
    int head, tail;
    int64_t begin, mine;
    DPB_D RowSplit(const T *row, int64_t vocab, int rank, int ranks)
    {
        const int off = misalignment(row);
        head = static_cast<int>(min(vocab, int64_t(off ? VEC - off : 0)));
        const int64_t all = (vocab - head) / VEC, each = (all + ranks - 1) / ranks;
        tail = static_cast<int>(vocab - head - all * VEC);
        begin = min(all, each * rank);
        mine = min(all, begin + each) - begin;
        if (rank > 0) head = 0;
        if (rank < ranks - 1) tail = 0;
    }
    // The thread's single element (head or tail), as a column; -1 without one.
    DPB_D int64_t single(int64_t vocab) const
    {
        const int t = threadIdx.x;
        return t < head ? t : t < head + tail ? vocab - tail + (t - head) : -1;
    }
};

// The gradient of the columns from the row's statistics: q = 2^((z - top) k - log2 of the sum), in which a row
// whose logits are all -inf counts as one of sum 1 (q is 0 then).
template <class T> struct RowGradient {
    using A = acc_t<T>;
    static constexpr bool ftz = is_half_v<T>;   // (float16 has no numbers as small as those that are flushed)
    A top, k, shift, g;
    DPB_D RowGradient(A top_, A log_sum, A k_, A g_)
        : top(SoftSum<A>::finite(top_)), k(k_), shift(log_sum == -INFINITY ? A(0) : -log_sum * A(kLog2E)), g(g_)
    {
    }
    DPB_D A q(A v) const { return exp2_<ftz>(fma_(v - top, k, shift)); }
    template <int N> DPB_D void apply(Values<A, N> &v) const
    {
        Values<A, N> e;
        e.fill(shift);
        v.add(-top);
        e.fma_add(v, k);
#pragma unroll
        for (int i = 0; i < N; ++i) v.set(i, exp2_<ftz>(e.get(i)));
        v.mul(g);
    }
};

// ------------------------------------------------------------------------------ rows in shared memory
// A cluster of 1 to 8 blocks takes a row and keeps it in its blocks' shared memory, so that the logits cross the
// memory once for loss and gradient: copies of all accesses are queued at once in four groups, each group is
// summed as it arrives (largest value and sum, both per thread), the blocks exchange their sums through
// distributed shared memory, and (GRAD) every block writes the gradient of its part.  The threads read only what
// they copied themselves, so that the copies need no barrier.
//
// Two exponentials an element: at float16 and the copy rate that is 3.3e12 a second, three quarters of what the
// special function units give; the rest of the arithmetic is done in pairs to stay out of their way.
constexpr int kGroups = 4;      // groups of copies
constexpr int kMaxRanks = 8;

template <class T, class I, bool GRAD>
__global__ void __launch_bounds__(512, 2)
    distillation_row_kernel(const T *z, RowMap zm, const acc_t<T> *top, const I *index, int k, int64_t vocab, acc_t<T> temp,
                            acc_t<T> inv_temp, acc_t<T> exp_scale, acc_t<T> *loss, acc_t<T> *stats, const acc_t<T> *dloss,
                            int64_t dstep, T *dz, RowMap dm, int ranks)
{
    using A = acc_t<T>;
    constexpr int VEC = vec_width<T>();
    using V = vec_t<T, VEC>;
    extern __shared__ __align__(16) char shared_bytes[];
    __shared__ SoftSum<A> warp_sums[16], rank_sums[kMaxRanks];
    __shared__ A buf[32], singles[2 * VEC];
    __shared__ int used;
    cudaGridDependencySynchronize();
    const uint32_t r = blockIdx.x / ranks;
    const int rank = blockIdx.x % ranks, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, threads = blockDim.x;
    const T *row = z + zm(r);
    const RowSplit<T> part(row, vocab, rank, ranks);
    const Teacher<A> teacher(shared_bytes, k);
    V *slot = reinterpret_cast<V *>(shared_bytes + (Teacher<A>::bytes(k) + 15) / 16 * 16);
    if (warp == 0) {
        const bool any = teacher.read(top + int64_t(r) * k, index + int64_t(r) * k, k, vocab);
        if (lane == 0) used = any;
    }
    __syncthreads();
    T *out = GRAD ? dz + dm(r) : nullptr;
    const int64_t first = part.begin * VEC + (rank == 0 ? part.head : misalignment(row) ? VEC - misalignment(row) : 0);
    const int64_t single = part.single(vocab);
    if (!used) {   // in every block of the cluster
        if (rank == 0 && threadIdx.x == 0) {
            if (loss) loss[r] = 0;
            if (stats) stats[2 * int64_t(r)] = stats[2 * int64_t(r) + 1] = 0;
        }
        if constexpr (GRAD) {
            const bool aligned = part.mine > 0 && misalignment(out + first) == 0;
            V zero;
#pragma unroll
            for (int j = 0; j < VEC; ++j) zero.v[j] = from_acc<T>(A(0));
            for (int64_t i = threadIdx.x; i < part.mine; i += threads) {
                T *o = out + first + i * VEC;
                if (aligned) *reinterpret_cast<V *>(o) = zero;
                else
#pragma unroll
                    for (int j = 0; j < VEC; ++j) o[j] = zero.v[j];
            }
            if (single >= 0) out[single] = zero.v[0];
        }
        return;
    }
    const int mine = static_cast<int>(part.mine), quarter = (mine + kGroups * threads - 1) / (kGroups * threads) * threads;
    const V *from = reinterpret_cast<const V *>(row + first);
    for (int g = 0; g < kGroups; ++g) {
        const int end = min(mine, (g + 1) * quarter);
        for (int i = g * quarter + threadIdx.x; i < end; i += threads) copy_async(slot + i, from + i);
        copy_async_commit();
    }
    const A alone = single >= 0 ? to_acc<A>(row[single]) : A(-INFINITY);
    if (single >= 0) singles[threadIdx.x] = alone;
    A *at_teacher = reinterpret_cast<A *>(slot + mine);   // the student's logits at the teacher's columns
    if (warp == 0) {
        if (rank == 0)   // (read before any block writes over them)
            for (int i = lane; i < k; i += 32)
                if (teacher.at[i] >= 0) at_teacher[i] = to_acc<A>(row[teacher.at[i]]);
        teacher.normalize(k, inv_temp);
    }
    SoftSum<A> s = {alone, single >= 0 && !(alone == -INFINITY) ? A(alone - alone + 1) : A(0)};
    const auto take = [&](int begin, int end) {
        constexpr int batch = 2;
        for (int i = begin + threadIdx.x; i < end; i += batch * threads) {
            Values<A, VEC> v[batch];
            unpack<A, VEC, T>(slot[i], v[0]);
            const bool more = i + threads < end;
            if (more) unpack<A, VEC, T>(slot[i + threads], v[1]);
            else v[1] = v[0];
            A best = v[0].get(0);
#pragma unroll
            for (int b = 0; b < batch; ++b)
#pragma unroll
                for (int j = 0; j < VEC; ++j) best = max_nan(best, v[b].get(j));
            s.raise(max_nan(s.top, best), exp_scale);
            const A down = -SoftSum<A>::finite(s.top);
#pragma unroll
            for (int b = 0; b < batch; ++b) {
                if (b > 0 && !more) break;
                v[b].add(down);
                v[b].mul(exp_scale);
                auto sum = Values<A, VEC>::all(0);
                Values<A, VEC> e;
#pragma unroll
                for (int j = 0; j < VEC; ++j) e.set(j, exp2_<true>(v[b].get(j)));
                e.sum_into(sum);
                s.sum += Values<A, VEC>::join(sum);
            }
        }
    };
    copy_async_wait<3>();
    take(0, min(mine, quarter));
    copy_async_wait<2>();
    take(quarter, min(mine, 2 * quarter));
    copy_async_wait<1>();
    take(2 * quarter, min(mine, 3 * quarter));
    copy_async_wait<0>();
    take(3 * quarter, mine);
    // lanes, warps and ranks, each in a fixed order
    s = s.over_warp(exp_scale);
    if (lane == 0) warp_sums[warp] = s;
    __syncthreads();
    s = lane < threads / 32 ? warp_sums[lane] : SoftSum<A>{-INFINITY, 0};
    s = s.over_warp(exp_scale);
    if (ranks > 1) {
        // every rank writes its sum to every rank; the barrier of the cluster makes them visible
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
        s = lane < ranks ? rank_sums[lane] : SoftSum<A>{-INFINITY, 0};
        s = s.over_warp(exp_scale);
    }
    const A log_sum = log_(s.sum);
    if (rank == 0) {
        A total = 0;
        for (int i = threadIdx.x; i < k; i += threads) {
            if (teacher.at[i] < 0 || teacher.p[i] == 0) continue;
            const A v = at_teacher[i];
            total += teacher.p[i] * (teacher.logp[i] - (v == -INFINITY ? A(-INFINITY) : (v - s.top) * inv_temp - log_sum));
        }
        total = block_fold(SumF(), total, buf);
        if (threadIdx.x == 0) {
            if (loss) loss[r] = temp * temp * total;
            if (stats) {
                stats[2 * int64_t(r)] = s.top;
                stats[2 * int64_t(r) + 1] = log_sum;
            }
        }
    }
    if constexpr (GRAD) {
        const RowGradient<T> grad(s.top, log_sum, exp_scale, dloss[r * dstep] * temp);
        const bool aligned = mine > 0 && misalignment(out + first) == 0;
        for (int i = threadIdx.x; i < mine; i += threads) {
            Values<A, VEC> v;
            unpack<A, VEC, T>(slot[i], v);
            grad.apply(v);
            const V w = repack<T, VEC, A>(v);
            T *o = out + first + int64_t(i) * VEC;
            if (aligned) *reinterpret_cast<V *>(o) = w;
            else
#pragma unroll
                for (int j = 0; j < VEC; ++j) o[j] = w.v[j];
        }
        if (single >= 0) out[single] = from_acc<T>(grad.g * grad.q(alone));
        __syncthreads();
        // the teacher's columns of this block's part once more, with its weight taken off
        const T *values = reinterpret_cast<const T *>(slot);
        for (int i = threadIdx.x; i < k; i += threads) {
            const int64_t c = teacher.at[i];
            if (c < 0) continue;
            const bool inside = c >= first && c < first + int64_t(mine) * VEC;
            if (!inside && !(c < part.head || c >= vocab - part.tail)) continue;
            A weight;
            if (!teacher.first_of_column(i, k, weight)) continue;
            if (inside) out[c] = from_acc<T>(grad.g * (grad.q(to_acc<A>(values[c - first])) - weight));
            else out[c] = from_acc<T>(grad.g * (grad.q(singles[c < part.head ? c : part.head + (c - (vocab - part.tail))]) - weight));
        }
    }
}

// ------------------------------------------------------------------------------------------ gradient alone
// From kept statistics: `ranks` blocks a row, each a part of it, four accesses of a thread in flight.
constexpr int kThreads = 256;

template <class T, class I>
__global__ void __launch_bounds__(kThreads)
    distillation_grad_kernel(const acc_t<T> *dloss, int64_t dstep, const T *z, RowMap zm, const acc_t<T> *top, const I *index, int k,
                             int64_t vocab, acc_t<T> temp, acc_t<T> inv_temp, acc_t<T> exp_scale, const acc_t<T> *stats, T *dz,
                             RowMap dm, int ranks)
{
    using A = acc_t<T>;
    constexpr int VEC = vec_width<T>(), flight = 4;
    using V = vec_t<T, VEC>;
    extern __shared__ __align__(16) char shared_bytes[];
    __shared__ int used;
    cudaGridDependencySynchronize();
    const uint32_t r = blockIdx.x / ranks;
    const int rank = blockIdx.x % ranks;
    const T *row = z + zm(r);
    T *out = dz + dm(r);
    const RowSplit<T> part(row, vocab, rank, ranks);
    const int64_t first = part.begin * VEC + (rank == 0 ? part.head : misalignment(row) ? VEC - misalignment(row) : 0);
    const int64_t last = first + part.mine * VEC, single = part.single(vocab);
    const Teacher<A> teacher(shared_bytes, k);
    A *at_teacher = reinterpret_cast<A *>(shared_bytes + (Teacher<A>::bytes(k) + 15) / 16 * 16);
    if (threadIdx.x < 32) {
        const bool any = teacher.read(top + int64_t(r) * k, index + int64_t(r) * k, k, vocab);
        if (threadIdx.x == 0) used = any;
        for (int i = threadIdx.x; i < k; i += 32) {   // before the block writes over them
            const int64_t c = teacher.at[i];
            const bool mine = c >= 0 && ((c >= first && c < last) || c < part.head || c >= vocab - part.tail);
            if (mine) at_teacher[i] = to_acc<A>(row[c]);
            else teacher.at[i] = c < 0 ? -1 : -2 - static_cast<int>(c);   // counts, in another block's part
        }
    }
    __syncthreads();
    const bool counts = used;
    const RowGradient<T> grad(counts ? stats[2 * int64_t(r)] : A(0), counts ? stats[2 * int64_t(r) + 1] : A(0), exp_scale,
                              dloss[r * dstep] * temp);
    const bool aligned = part.mine > 0 && misalignment(out + first) == 0;
    const auto put = [&](int64_t i, const V &w) {
        T *o = out + first + i * VEC;
        if (aligned) *reinterpret_cast<V *>(o) = w;
        else
#pragma unroll
            for (int j = 0; j < VEC; ++j) o[j] = w.v[j];
    };
    const V *from = reinterpret_cast<const V *>(row + first);
    V zero;
#pragma unroll
    for (int j = 0; j < VEC; ++j) zero.v[j] = from_acc<T>(A(0));
    for (int64_t i0 = threadIdx.x; i0 < part.mine; i0 += flight * kThreads) {
        V raw[flight];
#pragma unroll
        for (int f = 0; f < flight; ++f)
            if (counts && i0 + f * kThreads < part.mine) raw[f] = from[i0 + f * kThreads];
#pragma unroll
        for (int f = 0; f < flight; ++f) {
            if (i0 + f * kThreads >= part.mine) break;
            if (!counts) {
                put(i0 + f * kThreads, zero);
                continue;
            }
            Values<A, VEC> v;
            unpack<A, VEC, T>(raw[f], v);
            grad.apply(v);
            put(i0 + f * kThreads, repack<T, VEC, A>(v));
        }
    }
    if (single >= 0) out[single] = counts ? from_acc<T>(grad.g * grad.q(to_acc<A>(row[single]))) : zero.v[0];
    if (!counts) return;
    if (threadIdx.x < 32) {
        // all entries that count take part in the probabilities
        for (int i = threadIdx.x; i < k; i += 32)
            if (teacher.at[i] < -1) teacher.at[i] = -2 - teacher.at[i];
        __syncwarp();
        teacher.normalize(k, inv_temp);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < k; i += kThreads) {
        const int64_t c = teacher.at[i];
        if (c < 0 || !((c >= first && c < last) || c < part.head || c >= vocab - part.tail)) continue;
        A weight;
        if (teacher.first_of_column(i, k, weight)) out[c] = from_acc<T>(grad.g * (grad.q(at_teacher[i]) - weight));
    }
}

// Rows beyond the shared memory of a cluster: one block a row, read twice.
template <class T, class I>
__global__ void __launch_bounds__(1024)
    distillation_long_kernel(const T *z, RowMap zm, const acc_t<T> *top, const I *index, int k, int64_t vocab, acc_t<T> temp,
                             acc_t<T> inv_temp, acc_t<T> *loss, acc_t<T> *stats)
{
    using A = acc_t<T>;
    extern __shared__ __align__(16) char shared_bytes[];
    __shared__ A buf[3][32];
    __shared__ int used;
    const uint32_t r = blockIdx.x;
    const Teacher<A> teacher(shared_bytes, k);
    if (threadIdx.x < 32) {
        const bool any = teacher.read(top + int64_t(r) * k, index + int64_t(r) * k, k, vocab);
        if (any) teacher.normalize(k, inv_temp);
        if (threadIdx.x == 0) used = any;
    }
    __syncthreads();
    if (!used) {
        if (threadIdx.x == 0) {
            if (loss) loss[r] = 0;
            if (stats) stats[2 * int64_t(r)] = stats[2 * int64_t(r) + 1] = 0;
        }
        return;
    }
    const T *row = z + zm(r);
    A best = -INFINITY;
    for (int64_t c = threadIdx.x; c < vocab; c += blockDim.x) best = max_nan(best, to_acc<A>(row[c]));
    best = block_fold(MaxNanF(), best, buf[0]);
    A sum = 0;
    for (int64_t c = threadIdx.x; c < vocab; c += blockDim.x)
        sum += exp_((to_acc<A>(row[c]) - SoftSum<A>::finite(best)) * inv_temp);
    sum = block_fold(SumF(), sum, buf[1]);
    const A log_sum = log_(sum);
    A s = 0;
    for (int i = threadIdx.x; i < k; i += blockDim.x) {
        if (teacher.at[i] < 0 || teacher.p[i] == 0) continue;
        const A v = to_acc<A>(row[teacher.at[i]]);
        s += teacher.p[i] * (teacher.logp[i] - (v == -INFINITY ? A(-INFINITY) : (v - best) * inv_temp - log_sum));
    }
    s = block_fold(SumF(), s, buf[2]);
    if (threadIdx.x == 0) {
        if (loss) loss[r] = temp * temp * s;
        if (stats) {
            stats[2 * int64_t(r)] = best;
            stats[2 * int64_t(r) + 1] = log_sum;
        }
    }
}

// --------------------------------------------------------------------------------------- launchers
struct DistilArgs {
    const dpb_array *z, *top, *index, *dloss, *stats, *loss, *dz;
    RowMap zm, dm;
    int64_t rows, vocab, k;
    double temp;
};

template <class T, class I> static int run_grad(const DistilArgs &a, const acc_t<T> *stats, cudaStream_t s)
{
    using A = acc_t<T>;
    // a part of 64 KiB a block amortises the teacher's entries; few rows are split further
    const int64_t bytes = a.vocab * int64_t(sizeof(T));
    int64_t ranks = std::max<int64_t>(1, bytes / (64 * 1024));
    while (a.rows * ranks < 4 * device_props().sm_count && bytes / (2 * ranks) >= 8 * 1024) ranks *= 2;
    ranks = std::min<int64_t>(ranks, INT32_MAX / a.rows);
    launch_shared(distillation_grad_kernel<T, I>, static_cast<unsigned>(a.rows * ranks), unsigned(kThreads),
                  (Teacher<A>::bytes(int(a.k)) + 15) / 16 * 16 + size_t(a.k) * sizeof(A), s, static_cast<const A *>(a.dloss->data),
                  a.dloss->nd == 0 ? 0 : 1, static_cast<const T *>(a.z->data), a.zm, static_cast<const A *>(a.top->data),
                  static_cast<const I *>(a.index->data), static_cast<int>(a.k), a.vocab, A(a.temp), A(1.0 / a.temp),
                  A(kLog2E / a.temp), stats, static_cast<T *>(a.dz->data), a.dm, static_cast<int>(ranks));
    note_kernel("distillation_grad");
    return check_launch("distillation_grad");
}

template <class T, class I, bool GRAD> static int run_rows(const DistilArgs &a, int ranks, cudaStream_t s)
{
    using A = acc_t<T>;
    constexpr int VEC = vec_width<T>();
    const int64_t accesses = ceil_div(a.vocab / VEC, ranks);
    int threads = 64;   // eight accesses a thread
    while (threads < 512 && accesses > 8 * threads) threads *= 2;
    const size_t shared = (Teacher<A>::bytes(int(a.k)) + 15) / 16 * 16 + size_t(accesses) * 16 + size_t(a.k) * sizeof(A);
    launch_cluster(distillation_row_kernel<T, I, GRAD>, static_cast<unsigned>(a.rows * ranks), unsigned(ranks), unsigned(threads), shared, s,
                   static_cast<const T *>(a.z->data), a.zm, static_cast<const A *>(a.top->data),
                   static_cast<const I *>(a.index->data), static_cast<int>(a.k), a.vocab, A(a.temp), A(1.0 / a.temp),
                   A(kLog2E / a.temp), a.loss ? static_cast<A *>(a.loss->data) : nullptr,
                   a.stats ? static_cast<A *>(a.stats->data) : nullptr, GRAD ? static_cast<const A *>(a.dloss->data) : nullptr,
                   GRAD && a.dloss->nd > 0 ? 1 : 0, GRAD ? static_cast<T *>(a.dz->data) : nullptr, a.dm, ranks);
    note_kernel("distillation_row");
    return check_launch("distillation_row");
}

template <class T, class I> static int run_long(const DistilArgs &a, acc_t<T> *stats, cudaStream_t s)
{
    using A = acc_t<T>;
    distillation_long_kernel<T, I><<<static_cast<unsigned>(a.rows), 1024, Teacher<A>::bytes(int(a.k)), s>>>(
        static_cast<const T *>(a.z->data), a.zm, static_cast<const A *>(a.top->data), static_cast<const I *>(a.index->data),
        static_cast<int>(a.k), a.vocab, A(a.temp), A(1.0 / a.temp), a.loss ? static_cast<A *>(a.loss->data) : nullptr, stats);
    note_kernel("distillation_long");
    return check_launch("distillation_long");
}

// Blocks that share a row so that each holds at most 64 KiB (three blocks an SM are in different phases then); few
// rows are spread over more blocks as long as each has 8 KiB.  0: more than 8 blocks of 200 KiB.
static int row_ranks(int64_t rows, int64_t bytes)
{
    int ranks = 1;
    while (ranks < kMaxRanks && bytes > int64_t(ranks) * 64 * 1024) ranks *= 2;
    while (ranks < kMaxRanks && rows * ranks < 2 * device_props().sm_count && bytes / (2 * ranks) >= 8 * 1024) ranks *= 2;
    return bytes <= int64_t(ranks) * 200 * 1024 && rows <= INT32_MAX / ranks ? ranks : 0;
}

template <class T, class I> static int run(const DistilArgs &a, cudaStream_t s)
{
    using A = acc_t<T>;
    if (a.dz && !a.loss) return run_grad<T, I>(a, static_cast<const A *>(a.stats->data), s);
    const int ranks = row_ranks(a.rows, a.vocab * int64_t(sizeof(T)));
    if (ranks > 0) return a.dz ? run_rows<T, I, true>(a, ranks, s) : run_rows<T, I, false>(a, ranks, s);
    if (!a.dz) return run_long<T, I>(a, a.stats ? static_cast<A *>(a.stats->data) : nullptr, s);
    void *work = nullptr;
    DPB_TRY(dpb_malloc(static_cast<size_t>(2 * a.rows) * sizeof(A), s, &work));
    int st = run_long<T, I>(a, static_cast<A *>(work), s);
    if (st == DPB_OK) st = run_grad<T, I>(a, static_cast<const A *>(work), s);
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
