// Layer normalisation over the last axis and its gradient.
//
//   m = sum x / n,  r = 1 / sqrt(sum (x - m)^2 / n + eps),  h = (x - m) r,  y = h w + b
//   a = dy w,  dx = r (a - mean(a) - h mean(a h)),  dw = sum_rows dy h,  db = sum_rows dy
//
// Means, variances and all sums are float (double for float64 data); every result is rounded once.
// The variance is the mean of squared deviations from the mean (two sweeps over the row), not
// E[x^2] - m^2, which loses all digits of rows far from zero.  A sum overflows only where the mean itself
// does: every term of float32 and float64 data is divided by n as it is added (one multiplication, fused
// where it can be); float16 data cannot overflow a float32 sum.
#include "row_ops.cuh"

namespace dpb {

constexpr int kThreads = 256;

// --------------------------------------------------------------------------------------------- forward
// A group (a warp, or a block of as many warps as the row needs) takes R rows at a time, `step` rows apart, each
// thread the same columns of all rows.  What bounds such a kernel is the latency of the two folds a row
// and the instructions around them, not the bytes: R rows share the folds, and the arithmetic is done in
// pairs.  Rows are copied into shared memory ahead of their use (each thread its own accesses: no barrier),
// DEPTH - 1 rounds or, with one slot, from the moment that the rows before are in registers; that keeps 32 to
// 64 KiB an SM in flight.  The rows that are summed stay in registers as numbers of the accumulation type.
// Weight and bias are kept for all rows of a group, in registers or (KEEP = kShared) in the thread's own
// slots of shared memory: from L1 they cost more transfers than the data when they are float32 and the data
// float16.
constexpr int kGroupThreads = 1024;   // threads an SM, at 64 registers

enum Keep { kGlobal, kRegisters, kShared };

// Weight and bias of one thread's columns.
template <class W, int VEC, int ITEMS> struct KeptWeights {
    static constexpr int parts = VEC * sizeof(W) > 16 ? VEC * static_cast<int>(sizeof(W)) / 16 : 1;
    using S = vec_t<W, VEC / parts>;
    S *slot;       // [2][ITEMS][parts][threads]
    int threads;
    static size_t bytes(int threads) { return size_t(2) * ITEMS * parts * threads * sizeof(S); }
    DPB_D S &at(int which, int i, int k) const { return slot[((which * ITEMS + i) * parts + k) * threads]; }
    template <class RA> DPB_D void fill(int which, const W *w, const RA &ra, float otherwise) const
    {
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
#pragma unroll
            for (int k = 0; k < parts; ++k) {
                S v;
#pragma unroll
                for (int j = 0; j < VEC / parts; ++j) {
                    const int e = k * (VEC / parts) + j;
                    v.v[j] = w && ra.has(i, e) ? w[ra.column(i) + e] : from_acc<W>(acc_t<W>(otherwise));
                }
                at(which, i, k) = v;
            }
    }
    template <class A> DPB_D void get(int which, int i, Values<A, VEC> &out) const
    {
#pragma unroll
        for (int k = 0; k < parts; ++k) {
            Values<A, VEC / parts> some;
            unpack<A, VEC / parts, W>(at(which, i, k), some);
#pragma unroll
            for (int j = 0; j < VEC / parts; ++j) out.set(k * (VEC / parts) + j, some.get(j));
        }
    }
};

template <class T, class W, int VEC, int ITEMS, bool WARP, int R, int DEPTH, int KEEP, bool SHIFT>
__global__ void __launch_bounds__(WARP ? 256 : kGroupThreads, WARP ? kGroupThreads / 256 : 1)
    layer_norm_kernel(const T *x, RowMap xm, Span<T> xs, const W *w, const W *b, acc_t<T> eps, T *y, RowMap ym, acc_t<T> *mean,
                      acc_t<T> *rstd, uint32_t rows, int n)
{
    using A = acc_t<T>;
    using V = vec_t<T, VEC>;
    constexpr int groups = WARP ? 8 : 1;
    const int threads = WARP ? 256 : blockDim.x;
    extern __shared__ __align__(16) char shared_bytes[];
    __shared__ A buf[2][32 * R];
    if constexpr (!WARP) {
        for (int i = threadIdx.x; i < 2 * 32 * R; i += threads) (&buf[0][0])[i] = 0;
        __syncthreads();
    }
    cudaGridDependencySynchronize();
    const uint32_t step = gridDim.x * groups;
    uint32_t r = blockIdx.x * groups + (WARP ? threadIdx.x / 32 : 0);
    if (r >= rows) return;   // whole groups
    const RowAccess<T, VEC, ITEMS, SHIFT> at = {static_cast<int>(WARP ? threadIdx.x & 31 : threadIdx.x), WARP ? 32 : threads, n,
                                                SHIFT ? misalignment(x + xm(r)) : 0};
    V *slot = reinterpret_cast<V *>(shared_bytes) + threadIdx.x;   // [DEPTH][R][ITEMS][threads]
    at.clear(slot, threads, DEPTH * R);
    RowWalk<const T> xw(x, xm, r, step);
    RowWalk<T> yw(y, ym, r, step);
    uint32_t ahead = r;
    const auto fetch = [&](int to) {   // the next R rows into the ring
#pragma unroll
        for (int k = 0; k < R; ++k) {
            if (ahead >= rows) break;
            at.fetch(xw.p, slot + (to * R + k) * ITEMS * threads, threads, xs.lo, xs.hi);
            ahead += step;
            if (ahead < rows) xw.next(ahead);
        }
        copy_async_commit();
    };
    if constexpr (DEPTH == 1) fetch(0);
#pragma unroll
    for (int d = 0; d < DEPTH - 1; ++d) fetch(d);
    Values<A, VEC> wv[KEEP == kRegisters ? ITEMS : 1], bv[KEEP == kRegisters ? ITEMS : 1];
    using Kept = KeptWeights<W, VEC, ITEMS>;
    const Kept kept = {reinterpret_cast<typename Kept::S *>(shared_bytes + size_t(DEPTH) * R * ITEMS * threads * sizeof(V)) +
                           threadIdx.x,
                       threads};
    if constexpr (KEEP == kRegisters) {
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            at.load(w, i, wv[i], A(1));
            at.load(b, i, bv[i], A(0));
        }
    }
    else if constexpr (KEEP == kShared) {
        kept.fill(0, w, at, 1.0f);
        kept.fill(1, b, at, 0.0f);
    }
    bool edge[ITEMS];   // whether the warp has an access that reaches beyond the row
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) edge[i] = SHIFT && __any_sync(0xffffffffu, at.any(i) && !at.whole(i));
    const A inv_n = A(1) / A(n);
    int turn = 0;
    while (r < rows) {
        if constexpr (DEPTH > 1) fetch(turn == 0 ? DEPTH - 1 : turn - 1);
        copy_async_wait<DEPTH - 1>();
        Values<A, VEC> v[R][ITEMS];
        A m[R], rs[R];
#pragma unroll
        for (int k = 0; k < R; ++k) {
            auto sum = Values<A, VEC>::all(0);
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                unpack<A, VEC, T>(slot[((turn * R + k) * ITEMS + i) * threads], v[k][i]);
                if (SHIFT && edge[i]) at.clip(i, v[k][i]);
                if constexpr (is_half_v<T>) v[k][i].sum_into(sum);
                else v[k][i].sum_into(sum, inv_n);
            }
            m[k] = Values<A, VEC>::join(sum);
        }
        if constexpr (DEPTH == 1) fetch(0);   // the rows are in registers now
        turn = turn == DEPTH - 1 ? 0 : turn + 1;
        group_sums<WARP>(m, buf[0]);
#pragma unroll
        for (int k = 0; k < R; ++k) {
            if constexpr (is_half_v<T>) m[k] *= inv_n;
            auto sum = Values<A, VEC>::all(0);
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                v[k][i].add(at.any(i) ? -m[k] : A(0));   // zeros outside the row stay zeros
                if (SHIFT && edge[i]) at.clip(i, v[k][i]);
                if constexpr (is_half_v<T>) v[k][i].dot_into(sum, v[k][i]);
                else {
                    Values<A, VEC> d = v[k][i];
                    d.mul(inv_n);
                    d.dot_into(sum, v[k][i]);
                }
            }
            rs[k] = Values<A, VEC>::join(sum);
        }
        group_sums<WARP>(rs, buf[1]);
#pragma unroll
        for (int k = 0; k < R; ++k) {
            if (r >= rows) break;
            rs[k] = rsqrt_((is_half_v<T> ? rs[k] * inv_n : rs[k]) + eps);
            const bool aligned = !SHIFT || misalignment(yw.p) == at.mis;
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                if (!at.any(i)) continue;
                v[k][i].mul(rs[k]);
                Values<A, VEC> o, ww;
                if constexpr (KEEP == kRegisters) {
                    o = bv[i];
                    ww = wv[i];
                }
                else if constexpr (KEEP == kShared) {
                    kept.get(0, i, ww);
                    kept.get(1, i, o);
                }
                else {
                    at.load(w, i, ww, A(1));
                    at.load(b, i, o, A(0));
                }
                o.fma_add(v[k][i], ww);
                at.store(yw.p, i, repack<T, VEC, A>(o), aligned);
            }
            if (at.t == 0) {
                if (mean) mean[r] = m[k];
                if (rstd) rstd[r] = rs[k];
            }
            r += step;
            if (r < rows) yw.next(r);
        }
    }
}

// Rows too long for the registers of a block: read three times, the second and third time from L2.
template <class T, class W>
__global__ void __launch_bounds__(1024) layer_norm_long_kernel(const T *x, RowMap xm, const W *w, const W *b, acc_t<T> eps,
                                                               T *y, RowMap ym, acc_t<T> *mean, acc_t<T> *rstd, int64_t n)
{
    using A = acc_t<T>;
    __shared__ A buf[2][32];
    const uint32_t r = blockIdx.x;
    const T *xr = x + xm(r);
    T *yr = y + ym(r);
    const A inv_n = A(1) / A(n);
    A s = 0;
    for (int64_t c = threadIdx.x; c < n; c += blockDim.x) s = fma_(to_acc<A>(xr[c]), inv_n, s);
    const A m = block_fold(SumF(), s, buf[0]);
    s = 0;
    for (int64_t c = threadIdx.x; c < n; c += blockDim.x) {
        const A d = to_acc<A>(xr[c]) - m;
        s = fma_(d * inv_n, d, s);
    }
    const A rs = rsqrt_(block_fold(SumF(), s, buf[1]) + eps);
    for (int64_t c = threadIdx.x; c < n; c += blockDim.x) {
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

// One pass over dy and x for all three gradients.  The threads of a group own fixed columns, so that dw and
// db gather in registers over all rows of the group and one partial sum a block goes through memory; the
// rows travel through shared memory as in layer_norm_kernel.  HOLD: the products of the first sweep (dy w
// and h) stay in registers for the second and the ring has one slot; otherwise they are formed again from
// the ring.
template <class T, class W, int VEC, int ITEMS, bool WARP, int R, int DEPTH, bool HOLD, bool SHIFT, int THREADS>
__global__ void __launch_bounds__(WARP ? 256 : THREADS, WARP ? THREADS / 256 : 1)
    layer_norm_backward_kernel(const T *dy, RowMap dym, Span<T> dys, const T *x, RowMap xm, Span<T> xs, const acc_t<T> *mean,
                               const acc_t<T> *rstd, const W *w, T *dx, RowMap dxm, acc_t<T> *part, uint32_t rows, int n)
{
    static_assert(HOLD || DEPTH > 1, "the second sweep reads the ring");
    using A = acc_t<T>;
    using V = vec_t<T, VEC>;
    using Vals = Values<A, VEC>;
    constexpr int groups = WARP ? 8 : 1;
    const int threads = WARP ? 256 : blockDim.x;
    extern __shared__ __align__(16) char shared_bytes[];
    __shared__ A buf[2][32 * 2 * R];
    if constexpr (!WARP) {
        for (int i = threadIdx.x; i < 2 * 32 * 2 * R; i += threads) (&buf[0][0])[i] = 0;
        __syncthreads();
    }
    cudaGridDependencySynchronize();
    const uint32_t step = gridDim.x * groups;
    uint32_t r = blockIdx.x * groups + (WARP ? threadIdx.x / 32 : 0);
    const uint32_t first = r < rows ? r : 0;
    const RowAccess<T, VEC, ITEMS, SHIFT> at = {static_cast<int>(WARP ? threadIdx.x & 31 : threadIdx.x), WARP ? 32 : threads, n,
                                                SHIFT ? misalignment(x + xm(first)) : 0};
    V *slot = reinterpret_cast<V *>(shared_bytes) + threadIdx.x;   // [DEPTH][R][dy, x][ITEMS][threads]
    at.clear(slot, threads, DEPTH * R * 2);
    RowWalk<const T> gw(dy, dym, first, step), xw(x, xm, first, step);
    RowWalk<T> ow(dx, dxm, first, step);
    uint32_t ahead = r;
    const auto fetch = [&](int to) {
#pragma unroll
        for (int k = 0; k < R; ++k) {
            if (ahead >= rows) break;
            at.fetch(gw.p, slot + ((to * R + k) * 2) * ITEMS * threads, threads, dys.lo, dys.hi);
            at.fetch(xw.p, slot + ((to * R + k) * 2 + 1) * ITEMS * threads, threads, xs.lo, xs.hi);
            ahead += step;
            if (ahead < rows) {
                gw.next(ahead);
                xw.next(ahead);
            }
        }
        copy_async_commit();
    };
    if constexpr (DEPTH == 1) fetch(0);
#pragma unroll
    for (int d = 0; d < DEPTH - 1; ++d) fetch(d);
    using Kept = KeptWeights<W, VEC, ITEMS>;
    const Kept kept = {reinterpret_cast<typename Kept::S *>(shared_bytes + size_t(DEPTH) * R * 2 * ITEMS * threads * sizeof(V)) +
                           threadIdx.x,
                       threads};
    kept.fill(0, w, at, 1.0f);
    bool edge[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) edge[i] = SHIFT && __any_sync(0xffffffffu, at.any(i) && !at.whole(i));
    Vals dw[ITEMS], db[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        dw[i].fill(0);
        db[i].fill(0);
    }
    const A inv_n = A(1) / A(n);
    int turn = 0, fold = 0;
    A m_next[R], rs_next[R];
    const auto statistics = [&](uint32_t from) {   // of the next round's rows, ahead of their use
#pragma unroll
        for (int k = 0; k < R; ++k) {
            const uint32_t row = min(from + k * step, rows - 1);
            m_next[k] = mean[row];
            rs_next[k] = rstd[row];
        }
    };
    statistics(r);
    while (r < rows) {
        if constexpr (DEPTH > 1) fetch(turn == 0 ? DEPTH - 1 : turn - 1);
        A m[R], rs[R], s[2 * R];
#pragma unroll
        for (int k = 0; k < R; ++k) {
            m[k] = m_next[k];
            rs[k] = rs_next[k];
        }
        statistics(r + R * step);
        copy_async_wait<DEPTH - 1>();
        Vals a[HOLD ? R : 1][ITEMS], h[HOLD ? R : 1][ITEMS];
        // dy and h of a row from the ring
        const auto load = [&](int k, int i, Vals &aa, Vals &hh) {
            unpack<A, VEC, T>(slot[((turn * R + k) * 2 * ITEMS + i) * threads], aa);
            unpack<A, VEC, T>(slot[(((turn * R + k) * 2 + 1) * ITEMS + i) * threads], hh);
            hh.add(at.any(i) ? -m[k] : A(0));   // zeros outside the row stay zeros (m rs may be infinite)
            hh.mul(rs[k]);
            if (SHIFT && edge[i]) {
                at.clip(i, aa);
                at.clip(i, hh);
            }
        };
#pragma unroll
        for (int k = 0; k < R; ++k) {
            s[2 * k] = s[2 * k + 1] = 0;
            if (r + k * step >= rows) continue;   // nothing of the ring's older rows goes into dw and db
            auto sum1 = Vals::all(0), sum2 = sum1;
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                Vals &aa = a[HOLD ? k : 0][i], &hh = h[HOLD ? k : 0][i], ww;
                load(k, i, aa, hh);
                dw[i].fma_add(aa, hh);
                db[i].add(aa);
                kept.get(0, i, ww);
                aa.mul(ww);
                if constexpr (is_half_v<T>) {
                    aa.sum_into(sum1);
                    aa.dot_into(sum2, hh);
                }
                else {
                    Vals u = aa;
                    u.mul(inv_n);
                    u.sum_into(sum1);
                    u.dot_into(sum2, hh);
                }
            }
            s[2 * k] = Vals::join(sum1);
            s[2 * k + 1] = Vals::join(sum2);
        }
        if constexpr (DEPTH == 1) fetch(0);   // the rows are in registers now
        group_sums<WARP>(s, buf[fold]);
        fold ^= 1;
#pragma unroll
        for (int k = 0; k < R; ++k) {
            if (r >= rows) break;
            const A s1 = is_half_v<T> ? s[2 * k] * inv_n : s[2 * k], s2 = is_half_v<T> ? s[2 * k + 1] * inv_n : s[2 * k + 1];
            const bool aligned = !SHIFT || misalignment(ow.p) == at.mis;
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                if (!at.any(i)) continue;
                Vals &aa = a[HOLD ? k : 0][i], &hh = h[HOLD ? k : 0][i];
                if constexpr (!HOLD) {
                    Vals ww;
                    load(k, i, aa, hh);
                    kept.get(0, i, ww);
                    aa.mul(ww);
                }
                aa.add(-s1);
                aa.fma_add(hh, -s2);
                aa.mul(rs[k]);
                at.store(ow.p, i, repack<T, VEC, A>(aa), aligned);
            }
            r += step;
            if (r < rows) ow.next(r);
        }
        turn = turn == DEPTH - 1 ? 0 : turn + 1;
    }
    if (!part) return;
    part += int64_t(blockIdx.x) * 2 * n;
    if constexpr (WARP) {
        // the warps' sums, added in the order of the warps, over what was the ring
        copy_async_wait<0>();
        A *sum = reinterpret_cast<A *>(shared_bytes);
        for (int k = 0; k < groups; ++k) {
            __syncthreads();
            if (k != threadIdx.x / 32) continue;
#pragma unroll
            for (int i = 0; i < ITEMS; ++i)
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const int c = at.column(i) + j;
                    if (!at.has(i, j)) continue;
                    sum[c] = k ? sum[c] + dw[i].get(j) : dw[i].get(j);
                    sum[n + c] = k ? sum[n + c] + db[i].get(j) : db[i].get(j);
                }
        }
        __syncthreads();
        for (int c = threadIdx.x; c < 2 * n; c += threads) part[c] = sum[c];
    }
    else {
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const int c = at.column(i) + j;
                if (!at.has(i, j)) continue;
                part[c] = dw[i].get(j);
                part[n + c] = db[i].get(j);
            }
    }
}

// dw, db = sum of the partial sums: 64 columns a block, 32 threads a pair of columns that take every 32nd
// partial sum and are then added as a tree (one after the other they would lose what is small beside the first).
template <class A, class W>
__global__ void __launch_bounds__(1024) layer_norm_join_kernel(const A *part, int64_t slabs, int64_t n, W *dw, W *db)
{
    using P = typename pair_of<A>::type;
    __shared__ P buf[32][32];
    cudaGridDependencySynchronize();
    const int col = threadIdx.x & 31, lane = threadIdx.x >> 5;
    const int64_t i = (int64_t(blockIdx.x) * 32 + col) * 2;   // 2 n columns: pairs are whole and aligned
    P s = {0, 0};
    if (i < 2 * n) {
        const int64_t jump = 32 * n;   // pairs
        const P *p = reinterpret_cast<const P *>(part + lane * 2 * n + i);
        int64_t k = lane;
        for (; k + 7 * 32 < slabs; k += 8 * 32, p += 8 * jump) {   // eight loads in flight
            P v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) v[u] = p[u * jump];
#pragma unroll
            for (int u = 0; u < 8; ++u) s = add2(s, v[u]);
        }
        for (; k < slabs; k += 32, p += jump) s = add2(s, *p);
    }
    buf[lane][col] = s;
    __syncthreads();
    if (lane > 0 || i >= 2 * n) return;
    P t[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        P v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) v[u] = buf[8 * k + u][col];
#pragma unroll
        for (int d = 4; d > 0; d >>= 1)
#pragma unroll
            for (int u = 0; u < d; ++u) v[u] = add2(v[u], v[u + d]);
        t[k] = v[0];
    }
    s = add2(add2(t[0], t[1]), add2(t[2], t[3]));
    const auto put = [&](int64_t c, A v) { (c < n ? dw[c] : db[c - n]) = from_acc<W>(v); };
    put(i, s.x);
    put(i + 1, s.y);
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

// As many blocks as the SMs hold at once (limited by threads and by shared memory), but at least `rounds`
// rows a group.  Shifted rows: a group's rows have to start at one and the same misalignment, which a step
// of a multiple of 16 bytes' elements gives for rows one stride apart.
static unsigned block_count(int64_t rows, int groups, int rounds, int threads, size_t shared, bool shift, int an_sm_threads)
{
    const int64_t an_sm = std::max<int64_t>(1, std::min<int64_t>(an_sm_threads / threads, (227 * 1024) / int64_t(shared + 2048)));
    const int64_t most = device_props().sm_count * an_sm;
    int64_t blocks = std::min(most, ceil_div(rows, int64_t(groups) * rounds));
    if (shift && blocks * groups < rows) blocks = blocks < 8 ? 8 : blocks / 8 * 8;
    return static_cast<unsigned>(blocks);
}

// The elements of x for accesses that reach beyond a row; none when the rows are being overwritten.
template <class T> static Span<T> row_neighbours(const dpb_array &a, const dpb_array &out)
{
    const void *lo = nullptr, *hi = nullptr;
    if (a.data != out.data) array_bounds(a, lo, hi);
    return {static_cast<const T *>(lo), static_cast<const T *>(hi)};
}

template <class T, class W, int VEC, int ITEMS, bool WARP, int R, int DEPTH, int KEEP, bool SHIFT>
static bool launch_forward(const NormArgs &a, int64_t accesses, cudaStream_t s)
{
    using A = acc_t<T>;
    const int groups = WARP ? 8 : 1, threads = WARP ? 256 : static_cast<int>(ceil_div(ceil_div(accesses, ITEMS), 32) * 32);
    const size_t shared = size_t(DEPTH) * R * ITEMS * threads * sizeof(T) * VEC +
                          (KEEP == kShared ? KeptWeights<W, VEC, ITEMS>::bytes(threads) : 0);
    launch_shared<layer_norm_kernel<T, W, VEC, ITEMS, WARP, R, DEPTH, KEEP, SHIFT>>(
        block_count(a.rows, groups, 1, threads, shared, SHIFT, kGroupThreads), unsigned(threads), shared, s,
        static_cast<const T *>(a.x->data), a.xm, row_neighbours<T>(*a.x, *a.y),
        a.w ? static_cast<const W *>(a.w->data) : nullptr, a.b ? static_cast<const W *>(a.b->data) : nullptr, A(a.eps),
        static_cast<T *>(a.y->data), a.ym, a.mean ? static_cast<A *>(a.mean->data) : nullptr,
        a.rstd ? static_cast<A *>(a.rstd->data) : nullptr, static_cast<uint32_t>(a.rows), static_cast<int>(a.n));
    return true;
}

// Two accesses a thread and two rows at a time; measured at 32768 x 4096 float16 with float32 weights: 94 us
// (0.87 of the copy rate), against 106 us for one access and two rows, 126 us for two accesses and one row,
// 117 us for one access and four rows.  Weights: float16 rows of two accesses leave no registers for them
// (spills: 270 us), shared memory holds them; wider types keep them in registers.  Rows of at most 32
// accesses go to a warp (524288 x 256 float16: 104 us against 132 us), rows of more than 2048 take four
// accesses a thread and one row, with the weights in shared memory where they fit (4194 x 16001 float32: 103 us, 165 us
// from the caches).  So do shifted rows of more than 1024 accesses where two blocks fit an SM (16380 x 4097 float32:
// 94 us, 134 us with two accesses and 544 threads), and those of 65 to 128 accesses, for which one warp is enough then:
// 0.74 to 0.78 of the time of two warps and two rows up to 96 accesses and 0.83 to 0.97 above (111476 x 301 float32: 65 us
// against 86; 74565 x 225 float64: 55 against 66; 77582 x 865 float16: 86 against 90).  float16 rows with float32 weights
// are at 0.92 up to 96 accesses and at 1.12 above, where they stay with two warps.  False: the row is longer than 4096
// accesses.
template <class T, class W, int VEC, bool SHIFT> static bool run_rows(const NormArgs &a, cudaStream_t s)
{
    const int64_t nv = ceil_div(a.n + (SHIFT ? VEC - 1 : 0), VEC);
    if constexpr (VEC == 1) {   // single elements come eight at a time
        if (nv <= 256) return launch_forward<T, W, 1, 8, true, 1, 3, kRegisters, false>(a, nv, s);
        if (nv <= 8192) return launch_forward<T, W, 1, 8, false, 1, 3, kRegisters, false>(a, nv, s);
        return false;
    }
    else {
        constexpr int keep = is_half_v<T> ? kShared : kRegisters;
        if (nv <= 32) return launch_forward<T, W, VEC, 1, true, 2, 3, kRegisters, SHIFT>(a, nv, s);
        const int64_t four = ceil_div(ceil_div(nv, 4), 32) * 32 * 4 * VEC * (sizeof(T) + 2 * sizeof(W));   // bytes with four accesses
        constexpr int one_warp = sizeof(W) > sizeof(T) ? 96 : 128;
        if (SHIFT && ((nv > 64 && nv <= one_warp) || (nv > 1024 && nv <= 2048 && four <= 112 * 1024)))
            return launch_forward<T, W, VEC, 4, false, 1, 1, kShared, SHIFT>(a, nv, s);
        if (nv <= 2048) return launch_forward<T, W, VEC, 2, false, 2, 1, keep, SHIFT>(a, nv, s);
        if (nv <= 4096 && four <= 224 * 1024) return launch_forward<T, W, VEC, 4, false, 1, 1, kShared, SHIFT>(a, nv, s);
        if (nv <= 4096) return launch_forward<T, W, VEC, 4, false, 1, 2, kGlobal, SHIFT>(a, nv, s);
        return false;
    }
}

template <class T, class W> static int run_forward(const NormArgs &a, cudaStream_t s)
{
    using A = acc_t<T>;
    constexpr int wide = vec_width<T>();
    const W *w = a.w ? static_cast<const W *>(a.w->data) : nullptr, *b = a.b ? static_cast<const W *>(a.b->data) : nullptr;
    const bool aligned = row_vector(a.x->data, a.xm, a.n, sizeof(T), wide) == wide &&
                         row_vector(a.y->data, a.ym, a.n, sizeof(T), wide) == wide && wide_ok(w, wide, sizeof(W)) &&
                         wide_ok(b, wide, sizeof(W));
    const bool shifted = a.xm.one_stride();
    if (aligned ? run_rows<T, W, wide, false>(a, s)
                : shifted ? run_rows<T, W, wide, true>(a, s) : run_rows<T, W, 1, false>(a, s)) {
        note_kernel("layer_norm");
        return check_launch("layer_norm");
    }
    layer_norm_long_kernel<T, W><<<static_cast<unsigned>(a.rows), 1024, 0, s>>>(
        static_cast<const T *>(a.x->data), a.xm, w, b, A(a.eps), static_cast<T *>(a.y->data), a.ym,
        a.mean ? static_cast<A *>(a.mean->data) : nullptr, a.rstd ? static_cast<A *>(a.rstd->data) : nullptr, a.n);
    note_kernel("layer_norm_long");
    return check_launch("layer_norm_long");
}

struct NormGradArgs {
    const dpb_array *dy, *x, *mean, *rstd, *w, *dx, *dw, *db;
    RowMap dym, xm, dxm;
    int64_t rows, n;
};

template <class T, class W> static int join_partials(const NormGradArgs &a, const acc_t<T> *part, int64_t slabs, cudaStream_t s)
{
    launch_after_previous(layer_norm_join_kernel<acc_t<T>, W>, static_cast<unsigned>(ceil_div(a.n, 32)), 1024u, s, part,
                          slabs, a.n, static_cast<W *>(a.dw->data), static_cast<W *>(a.db->data));
    note_kernel("layer_norm_join");
    return check_launch("layer_norm_join");
}

template <class T, class W, int VEC, int ITEMS, bool WARP, int R, int DEPTH, bool HOLD, bool SHIFT, int THREADS>
static int launch_backward(const NormGradArgs &a, int64_t accesses, cudaStream_t s)
{
    using A = acc_t<T>;
    const int groups = WARP ? 8 : 1, threads = WARP ? 256 : static_cast<int>(ceil_div(ceil_div(accesses, ITEMS), 32) * 32);
    // (half of what KeptWeights keeps: there is no bias)
    const size_t shared = size_t(DEPTH) * R * 2 * ITEMS * threads * sizeof(T) * VEC + KeptWeights<W, VEC, ITEMS>::bytes(threads) / 2;
    const unsigned blocks = block_count(a.rows, groups, R, threads, shared, SHIFT, THREADS);
    void *part = nullptr;
    if (a.dw) DPB_TRY(dpb_malloc(static_cast<size_t>(int64_t(blocks) * 2 * a.n) * sizeof(A), s, &part));
    launch_shared<layer_norm_backward_kernel<T, W, VEC, ITEMS, WARP, R, DEPTH, HOLD, SHIFT, THREADS>>(
        blocks, unsigned(threads), shared, s, static_cast<const T *>(a.dy->data), a.dym, row_neighbours<T>(*a.dy, *a.dx),
        static_cast<const T *>(a.x->data), a.xm, row_neighbours<T>(*a.x, *a.dx), static_cast<const A *>(a.mean->data),
        static_cast<const A *>(a.rstd->data), a.w ? static_cast<const W *>(a.w->data) : nullptr,
        static_cast<T *>(a.dx->data), a.dxm, static_cast<A *>(part), static_cast<uint32_t>(a.rows), static_cast<int>(a.n));
    note_kernel("layer_norm_backward");
    int st = check_launch("layer_norm_backward");
    if (part) {
        if (st == DPB_OK) st = join_partials<T, W>(a, static_cast<const A *>(part), blocks, s);
        dpb_free(part, s);
    }
    return st;
}

// Measured at 16384 x 4096 float16 with float32 weights and 8192 x 4096 float32 (us):
//   1024 threads an SM, one access, one row:  97 / 78; two rows: 105 / 76;
//   512 threads an SM, two accesses, one row: 95 / 82; two rows: 96 / 74 (92 / 74 at 2048 columns).
// More accesses a thread cost fewer instructions around the folds, fewer threads leave 128 registers for the
// accumulators.  Shifted rows of float16 need registers for the edges too: one row, 640 threads.
// Shifted rows of other types just above 1024 accesses take four, so that two blocks fit an SM (16380 x 4097 float32: 156
// us against 240 with one block of 544 threads; at 6001 columns that form is slower, 226 against 197).
// False: the row is too long (then the columns are summed by a second pass over dy and x).
template <class T, class W, int VEC, bool SHIFT> static bool run_rows_backward(const NormGradArgs &a, cudaStream_t s, int &st)
{
    const int64_t nv = ceil_div(a.n + (SHIFT ? VEC - 1 : 0), VEC);
#define DPB_BACK(LIMIT, ITEMS, WARP, R, DEPTH, HOLD, THREADS)                                                       \
    if (nv <= (LIMIT)) {                                                                                            \
        st = launch_backward<T, W, VEC, ITEMS, WARP, R, DEPTH, HOLD, SHIFT, THREADS>(a, nv, s);                     \
        return true;                                                                                                \
    }
    if constexpr (VEC == 1) {
        DPB_BACK(128, 4, true, 1, 3, true, 1024)
        DPB_BACK(4096, 4, false, 1, 2, true, 1024)
    }
    else {
        DPB_BACK(32, 1, true, 2, 2, false, 1024)
        if constexpr (!is_half_v<T>) {
            DPB_BACK(1024, 2, false, 2, 1, true, 512)
        }
        else if constexpr (SHIFT) {
            DPB_BACK(1280, 2, false, 1, 2, true, 640)
        }
        else {
            DPB_BACK(1024, 2, false, 2, 2, false, 512)
        }
        if constexpr (SHIFT && !is_half_v<T>) {
            DPB_BACK(1280, 4, false, 1, 2, false, 640)
        }
        if constexpr (SHIFT) {
            DPB_BACK(2048, 2, false, 1, 2, false, 1024)
        }
        else {
            DPB_BACK(2048, 4, false, 1, 2, false, 512)
        }
    }
#undef DPB_BACK
    return false;
}

template <class T, class W> static int run_backward(const NormGradArgs &a, cudaStream_t s)
{
    using A = acc_t<T>;
    const T *dy = static_cast<const T *>(a.dy->data), *x = static_cast<const T *>(a.x->data);
    const A *mean = static_cast<const A *>(a.mean->data), *rstd = static_cast<const A *>(a.rstd->data);
    const W *w = a.w ? static_cast<const W *>(a.w->data) : nullptr;
    constexpr int wide = vec_width<T>();
    if (a.rows > 0) {
        const bool aligned = row_vector(x, a.xm, a.n, sizeof(T), wide) == wide &&
                             row_vector(dy, a.dym, a.n, sizeof(T), wide) == wide &&
                             row_vector(a.dx->data, a.dxm, a.n, sizeof(T), wide) == wide;
        // shifted columns: rows one stride apart that start at the same misalignment in dy and x
        const bool shifted = (a.rows == 1 || (a.xm.one_stride() && a.dym.one_stride() && (a.xm.inner - a.dym.inner) % wide == 0)) &&
                             (reinterpret_cast<uintptr_t>(x) - reinterpret_cast<uintptr_t>(dy)) % 16 == 0;
        int st = DPB_OK;
        if (aligned ? run_rows_backward<T, W, wide, false>(a, s, st)
                    : shifted ? run_rows_backward<T, W, wide, true>(a, s, st) : run_rows_backward<T, W, 1, false>(a, s, st))
            return st;
    }
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
        int st = check_launch("layer_norm_columns");
        if (st == DPB_OK) st = join_partials<T, W>(a, static_cast<const A *>(part), slabs, s);
        dpb_free(part, s);
        DPB_TRY(st);
    }
    if (a.rows == 0) return DPB_OK;
    layer_norm_dx_kernel<T, W><<<static_cast<unsigned>(a.rows), kThreads, 0, s>>>(dy, a.dym, x, a.xm, mean, rstd, w,
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
