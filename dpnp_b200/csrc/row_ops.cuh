// Shared parts of the row operators (layer normalisation, embedding lookup, distillation loss):
// how the rows of a descriptor lie in memory, accumulation types, block-wide sums, and the argument
// checks of their entry points.
#pragma once

#include <atomic>
#include <cmath>
#include <initializer_list>
#include <vector>

#include "common.cuh"
#include "iterspace.h"

namespace dpb {

// Sums and statistics are held in float for float16 and float32 data, in double for float64.
template <class T> struct acc_of { using type = float; };
template <> struct acc_of<double> { using type = double; };
template <class T> using acc_t = typename acc_of<T>::type;
inline int acc_typenum(int tn) { return tn == DPB_DOUBLE ? DPB_DOUBLE : DPB_FLOAT; }

template <class A, class T> DPB_D A to_acc(T v)
{
    if constexpr (is_half_v<T>) return __half2float(v);
    else return static_cast<A>(v);
}
// The one rounding of a result to its element type (to nearest even).
template <class T, class A> DPB_D T from_acc(A v)
{
    if constexpr (is_half_v<T>) return __float2half_rn(v);
    else return static_cast<T>(v);
}

// Element offset of row r: the leading axes of an array, collapsed to at most two levels.
struct RowMap {
    int64_t outer, inner;   // strides of the two levels in elements
    FastDiv32 extent;       // rows of one inner level
    bool nested = false;    // two levels (whatever their strides are: an outer one of 0 is a broadcast axis)
    DPB_HD bool one_stride() const { return !nested; }   // all rows are `inner` apart
    DPB_HD int64_t operator()(uint32_t r) const
    {
        uint32_t q, m;
        extent.divmod(r, q, m);
        return int64_t(q) * outer + int64_t(m) * inner;
    }
};

// Walks rows r, r + step, r + 2 step, ... of an array: an addition a row where they are one stride apart.
template <class T> struct RowWalk {
    T *base, *p;
    RowMap map;
    int64_t delta;
    DPB_HD RowWalk(T *data, const RowMap &m, uint32_t r, uint32_t step)
        : base(data), p(data + m(r)), map(m), delta(m.one_stride() ? int64_t(step) * m.inner : 0)
    {
    }
    DPB_HD void next(uint32_t r)   // to row r, one step on (r < 2^31: the caller does not go beyond the last row)
    {
        if (map.one_stride()) p += delta;
        else p = base + map(r);
    }
};

// Host: rows of `a` (its leading nd-1 axes) as a RowMap; false when the last axis is not unit-stride
// or the leading axes need more than two levels.
inline bool make_row_map(const dpb_array &a, RowMap &map)
{
    const int lead = a.nd - 1;
    const std::vector<int64_t> st = strides_of(a);
    if (a.shape[lead] > 1 && st[lead] != 1) return false;
    int64_t ext[2] = {1, 1}, str[2] = {0, 0};
    int levels = 0;
    for (int i = 0; i < lead; ++i) {
        if (a.shape[i] == 1) continue;
        if (levels > 0 && str[levels - 1] == st[i] * a.shape[i]) {
            ext[levels - 1] *= a.shape[i];
            str[levels - 1] = st[i];
            continue;
        }
        if (levels == 2) return false;
        ext[levels] = a.shape[i];
        str[levels] = st[i];
        ++levels;
    }
    map.nested = levels == 2;
    if (map.nested) {
        map.outer = str[0];
        map.inner = str[1];
        map.extent = FastDiv32(static_cast<uint32_t>(ext[1]));
    }
    else {
        map.outer = 0;
        map.inner = str[0];
        map.extent = FastDiv32(static_cast<uint32_t>(ext[0] > 0 ? ext[0] : 1));
    }
    return true;
}

// Largest power-of-two number of elements (at most `most`) that divides every row start and the
// width, i.e. the widest access with which all rows can be walked.
inline int row_vector(const void *p, const RowMap &map, int64_t width, int item, int most)
{
    int v = most;
    while (v > 1 && (!is_aligned(p, static_cast<size_t>(v) * item) || map.outer % v || map.inner % v || width % v)) v /= 2;
    return v;
}

// The same for an operand that is read with the rows (a weight): its accesses are of 16 bytes at most.
inline bool wide_ok(const void *p, int vec, int item)
{
    const int bytes = vec * item;
    return !p || is_aligned(p, static_cast<size_t>(bytes > 16 ? 16 : bytes));
}

// Lets a kernel have as much dynamic shared memory as a block can (more than 48 KiB in all have to be asked for).  The limit
// belongs to the function on the device and all threads of the program share it: it is raised once and stays, because a
// limit set to each call's own size could be lowered by another thread before the launch.  False: an error, which is left in
// cudaGetLastError.
template <auto kernel> inline bool allow_shared()
{
    static std::atomic<uint64_t> done{0};   // a bit a device
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return false;
    const uint64_t bit = uint64_t(1) << (dev & 63);
    if (dev < 64 && (done.load(std::memory_order_acquire) & bit)) return true;
    cudaFuncAttributes has;
    if (cudaFuncGetAttributes(&has, kernel) != cudaSuccess ||
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             device_props().max_smem_optin - static_cast<int>(has.sharedSizeBytes)) != cudaSuccess)
        return false;
    if (dev < 64) done.fetch_or(bit, std::memory_order_release);
    return true;
}

template <class... KArgs, class... Args> inline void launch_config(const cudaLaunchConfig_t &cfg, void (*kernel)(KArgs...), Args... args)
{
    cudaLaunchKernelEx(&cfg, kernel, KArgs(args)...);   // an error stays in cudaGetLastError for check_launch
}

// launch_after_previous with dynamic shared memory and clusters of `cluster` blocks.
template <auto kernel, class... Args>
inline void launch_cluster(unsigned grid, unsigned cluster, unsigned block, size_t shared, cudaStream_t stream, Args... args)
{
    if (shared > 40 * 1024 && !allow_shared<kernel>()) return;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = shared;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    if (tuning_pdl()) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (cluster > 1) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attr[cfg.numAttrs].val.clusterDim.x = cluster;
        attr[cfg.numAttrs].val.clusterDim.y = 1;
        attr[cfg.numAttrs++].val.clusterDim.z = 1;
    }
    cfg.attrs = attr;
    launch_config(cfg, kernel, args...);
}
template <auto kernel, class... Args>
inline void launch_shared(unsigned grid, unsigned block, size_t shared, cudaStream_t stream, Args... args)
{
    launch_cluster<kernel>(grid, 1u, block, shared, stream, args...);
}

// -------------------------------------------------------------------------------- argument checks
constexpr int64_t kMaxRows = INT32_MAX;   // row numbers are divided with 31-bit arithmetic

// First element of an array and the one behind its last.
inline void array_bounds(const dpb_array &a, const void *&lo, const void *&hi)
{
    int64_t first, last;
    displacement_range(a, first, last);
    const char *p = static_cast<const char *>(a.data);
    lo = p + first * type_size(a.typenum);
    hi = p + (last + 1) * type_size(a.typenum);
}

inline int64_t count_rows(const dpb_array &a)
{
    int64_t n = 1;
    for (int i = 0; i + 1 < a.nd; ++i) n *= a.shape[i];
    return n;
}

// A descriptor that is valid in itself and whose elements lie on their own alignment.
inline int check_operand(const dpb_array *a, const char *what)
{
    DPB_TRY(check_array(a, what));
    if (num_elements(*a) > 0 && (!a->data || !is_aligned(a->data, type_size(a->typenum) > 8 ? 8 : type_size(a->typenum))))
        return set_error(DPB_ERR_VALUE, "%s: null or misaligned data pointer", what);
    return DPB_OK;
}

inline int check_float_type(const dpb_array &a, const char *what)
{
    if (a.typenum != DPB_HALF && a.typenum != DPB_FLOAT && a.typenum != DPB_DOUBLE)
        return set_error(DPB_ERR_TYPE, "%s: float16, float32 or float64 is needed, got %s", what, type_name(a.typenum));
    return DPB_OK;
}

inline int check_type(const dpb_array &a, int tn, const char *what)
{
    if (a.typenum != tn)
        return set_error(DPB_ERR_VALUE, "%s: type %s is needed, got %s", what, type_name(tn), type_name(a.typenum));
    return DPB_OK;
}

// Device, writability and no element written twice.
inline int check_output(const dpb_array &a, const char *what)
{
    if (!(a.flags & DPB_FLAG_WRITABLE)) return set_error(DPB_ERR_VALUE, "%s: output array is read-only.", what);
    const std::vector<int64_t> st = strides_of(a);
    int64_t lo, hi;
    displacement_range(a, lo, hi);
    const int64_t n = num_elements(a);
    bool twice = hi - lo + 1 < n;
    for (int i = 0; i < a.nd; ++i) twice = twice || (n > 0 && a.shape[i] > 1 && st[i] == 0);
    if (twice)
        return set_error(DPB_ERR_VALUE, "%s: Memory addressed by the output array is not sufficiently ample.", what);
    return DPB_OK;
}

inline int check_same_device(const dpb_array &a, const dpb_array &b)
{
    if (a.device != b.device)
        return set_error(DPB_ERR_VALUE, "Execution queue is not compatible with allocation queues");
    return DPB_OK;
}

// Shape `lead[0..nlead)` followed by `tail` (tail < 0: nothing follows).
inline int check_shape(const dpb_array &a, const int64_t *lead, int nlead, int64_t tail, const char *what)
{
    bool ok = a.nd == nlead + (tail >= 0 ? 1 : 0);
    for (int i = 0; ok && i < nlead; ++i) ok = a.shape[i] == lead[i];
    if (ok && tail >= 0) ok = a.shape[nlead] == tail;
    if (!ok) return set_error(DPB_ERR_VALUE, "%s: shape does not match the other arrays", what);
    return DPB_OK;
}

inline bool is_c_contiguous(const dpb_array &a)
{
    const std::vector<int64_t> st = strides_of(a);
    int64_t acc = 1;
    for (int i = a.nd - 1; i >= 0; --i) {
        if (a.shape[i] == 0) return true;
        if (a.shape[i] != 1 && st[i] != acc) return false;
        acc *= a.shape[i];
    }
    return true;
}

inline int check_c_contiguous(const dpb_array &a, const char *what)
{
    if (!is_c_contiguous(a)) return set_error(DPB_ERR_VALUE, "%s: a C-contiguous array is needed", what);
    return DPB_OK;
}

inline int check_row_map(const dpb_array &a, RowMap &map, const char *what)
{
    if (!make_row_map(a, map))
        return set_error(DPB_ERR_VALUE, "%s: rows of unit stride, at most two levels apart, are needed", what);
    return DPB_OK;
}

// `out` may be exactly one of the arrays it is computed from (each row or element is read before it
// is written) where `in_place` says so; any other overlap is refused.
inline int check_no_overlap(const dpb_array &in, const dpb_array &out, bool in_place)
{
    if (arrays_overlap(in, out) && !(in_place && same_logical_tensors(in, out)))
        return set_error(DPB_ERR_VALUE, "Arrays index overlapping segments of memory");
    return DPB_OK;
}

// No output overlaps an input or another output (null pointers: absent arrays).
inline int check_no_overlaps(std::initializer_list<const dpb_array *> in, std::initializer_list<const dpb_array *> out)
{
    for (auto o = out.begin(); o != out.end(); ++o) {
        if (!*o) continue;
        for (const dpb_array *i : in)
            if (i) DPB_TRY(check_no_overlap(*i, **o, false));
        for (auto p = out.begin(); p != o; ++p)
            if (*p) DPB_TRY(check_no_overlap(**p, **o, false));
    }
    return DPB_OK;
}

// --------------------------------------------------------------------------------- block-wide folds
struct SumF {
    template <class A> DPB_D A operator()(A a, A b) const { return a + b; }
};
struct MaxF {   // a NaN stays a NaN
    template <class A> DPB_D A operator()(A a, A b) const { return (a > b || a != a) ? a : b; }
};

template <class F, class A> DPB_D A warp_fold(F f, A v)
{
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, d));
    return v;
}

// Fold over the block in a fixed order; every thread gets the result.  `buf` holds one value per warp
// and may be used again after the next __syncthreads().
template <class F, class A> DPB_D A block_fold(F f, A v, A *buf)
{
    const int nwarp = blockDim.x >> 5;
    v = warp_fold(f, v);
    if (nwarp == 1) return v;
    if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
    __syncthreads();
    v = buf[0];
    for (int w = 1; w < nwarp; ++w) v = f(v, buf[w]);
    return v;
}

// R sums (R = 1, 2 or 4) over a warp (WARP) or over the whole block, the same bits in every thread.  The
// first steps of the folds hand each half (quarter) of the warp one sum to go on with, which saves
// shuffles; one barrier where there are several warps.  `buf` (32 R values, zeros where the block has no
// warp) must not be the one of the previous call: slower threads may still be reading that.
template <bool WARP, int R, class A> DPB_D void group_sums(A (&v)[R], A *buf)
{
    constexpr unsigned all = 0xffffffffu;
    constexpr int part = 32 / R;   // lanes that share a sum
    const int lane = threadIdx.x & 31;
    A s = v[0];
    if constexpr (R == 2) {
        const bool low = lane < 16;
        s = (low ? v[0] : v[1]) + __shfl_xor_sync(all, low ? v[1] : v[0], 16);
    }
    else if constexpr (R == 4) {
        const bool low = lane < 16, even = (lane & 8) == 0;
        const A p = (low ? v[0] : v[2]) + __shfl_xor_sync(all, low ? v[2] : v[0], 16);
        const A q = (low ? v[1] : v[3]) + __shfl_xor_sync(all, low ? v[3] : v[1], 16);
        s = (even ? p : q) + __shfl_xor_sync(all, even ? q : p, 8);
    }
#pragma unroll
    for (int d = part / 2; d > 0; d >>= 1) s += __shfl_xor_sync(all, s, d);
    if constexpr (!WARP) {
        A *mine = buf + lane / part * 32;
        const int at = lane & (part - 1);
        if (at == 0) mine[threadIdx.x >> 5] = s;
        __syncthreads();
        s = mine[at];
#pragma unroll
        for (int k = part; k < 32; k += part) s += mine[k + at];
#pragma unroll
        for (int d = part / 2; d > 0; d >>= 1) s += __shfl_xor_sync(all, s, d);
    }
    if constexpr (R == 1) v[0] = s;
    else {
#pragma unroll
        for (int k = 0; k < R; ++k) v[k] = __shfl_sync(all, s, k * part);
    }
}

// fmaf / fma under the library's -fmad=false
DPB_D float fma_(float a, float b, float c) { return fmaf(a, b, c); }
DPB_D double fma_(double a, double b, double c) { return fma(a, b, c); }
DPB_D float exp_(float a) { return expf(a); }
DPB_D double exp_(double a) { return exp(a); }
DPB_D float log_(float a) { return logf(a); }
DPB_D double log_(double a) { return log(a); }
// 1 / sqrt(a): within 2 steps of float, 1 of double; a quotient and a root cost ten times the instructions
DPB_D float rsqrt_(float a) { return rsqrtf(a); }
DPB_D double rsqrt_(double a) { return rsqrt(a); }

// ----------------------------------------------------------------------------- arrays in registers
// Element-wise arithmetic on a thread's values.  float pairs go through the two-lane instructions
// (add/mul/fma.rn.f32x2, each lane rounded as the scalar instruction rounds it), which halves the
// number of instructions: with 16-bit data these kernels are otherwise bound by issue, not by memory.
DPB_D float2 add2(float2 a, float2 b)
{
    float2 r;
    asm("add.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<unsigned long long &>(r))
        : "l"(reinterpret_cast<unsigned long long &>(a)), "l"(reinterpret_cast<unsigned long long &>(b)));
    return r;
}
DPB_D float2 mul2(float2 a, float2 b)
{
    float2 r;
    asm("mul.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<unsigned long long &>(r))
        : "l"(reinterpret_cast<unsigned long long &>(a)), "l"(reinterpret_cast<unsigned long long &>(b)));
    return r;
}
DPB_D float2 fma2(float2 a, float2 b, float2 c)
{
    float2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(reinterpret_cast<unsigned long long &>(r))
        : "l"(reinterpret_cast<unsigned long long &>(a)), "l"(reinterpret_cast<unsigned long long &>(b)),
          "l"(reinterpret_cast<unsigned long long &>(c)));
    return r;
}
DPB_D double2 add2(double2 a, double2 b) { return make_double2(a.x + b.x, a.y + b.y); }
DPB_D double2 mul2(double2 a, double2 b) { return make_double2(a.x * b.x, a.y * b.y); }
DPB_D double2 fma2(double2 a, double2 b, double2 c) { return make_double2(fma(a.x, b.x, c.x), fma(a.y, b.y, c.y)); }
template <class A> struct pair_of { using type = float2; };
template <> struct pair_of<double> { using type = double2; };

// N values as N / 2 pairs (N even) or single values.
template <class A, int N> struct Values {
    static constexpr bool paired = N % 2 == 0;
    using P = std::conditional_t<paired, typename pair_of<A>::type, A>;
    static constexpr int M = paired ? N / 2 : N;
    P p[M];
    static DPB_D P all(A s)
    {
        if constexpr (paired) return P{s, s};
        else return s;
    }
    static DPB_D P add_(P a, P b)
    {
        if constexpr (paired) return add2(a, b);
        else return a + b;
    }
    static DPB_D P mul_(P a, P b)
    {
        if constexpr (paired) return mul2(a, b);
        else return a * b;
    }
    static DPB_D P fma3(P a, P b, P c)
    {
        if constexpr (paired) return fma2(a, b, c);
        else return fma_(a, b, c);
    }
    DPB_D A get(int i) const
    {
        if constexpr (paired) return i & 1 ? p[i / 2].y : p[i / 2].x;
        else return p[i];
    }
    DPB_D void set(int i, A v)
    {
        if constexpr (paired) (i & 1 ? p[i / 2].y : p[i / 2].x) = v;
        else p[i] = v;
    }
    DPB_D void fill(A s)
    {
#pragma unroll
        for (int i = 0; i < M; ++i) p[i] = all(s);
    }
    DPB_D void add(const Values &o)   // += o
    {
#pragma unroll
        for (int i = 0; i < M; ++i) p[i] = add_(p[i], o.p[i]);
    }
    DPB_D void add(A s)
    {
#pragma unroll
        for (int i = 0; i < M; ++i) p[i] = add_(p[i], all(s));
    }
    DPB_D void mul(const Values &o)
    {
#pragma unroll
        for (int i = 0; i < M; ++i) p[i] = mul_(p[i], o.p[i]);
    }
    DPB_D void mul(A s)
    {
#pragma unroll
        for (int i = 0; i < M; ++i) p[i] = mul_(p[i], all(s));
    }
    DPB_D void fma_add(const Values &a, const Values &b)   // += a b
    {
#pragma unroll
        for (int i = 0; i < M; ++i) p[i] = fma3(a.p[i], b.p[i], p[i]);
    }
    DPB_D void fma_add(const Values &a, A s)   // += a s
    {
#pragma unroll
        for (int i = 0; i < M; ++i) p[i] = fma3(a.p[i], all(s), p[i]);
    }
    // sums that gather in one pair (one value): one instruction a pair, then a single addition
    DPB_D void sum_into(P &s) const
    {
#pragma unroll
        for (int i = 0; i < M; ++i) s = add_(s, p[i]);
    }
    DPB_D void sum_into(P &s, A times) const
    {
#pragma unroll
        for (int i = 0; i < M; ++i) s = fma3(p[i], all(times), s);
    }
    DPB_D void dot_into(P &s, const Values &o) const
    {
#pragma unroll
        for (int i = 0; i < M; ++i) s = fma3(p[i], o.p[i], s);
    }
    static DPB_D A join(P s)
    {
        if constexpr (paired) return s.x + s.y;
        else return s;
    }
};

// VEC stored elements to numbers of the accumulation type and back (each rounded once).
template <class A, int N, class T> DPB_D void unpack(const vec_t<T, N> &v, Values<A, N> &out)
{
    if constexpr (is_half_v<T> && N % 2 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 2) out.p[i / 2] = __half22float2(*reinterpret_cast<const __half2 *>(v.v + i));
    }
    else {
#pragma unroll
        for (int i = 0; i < N; ++i) out.set(i, to_acc<A>(v.v[i]));
    }
}
template <class T, int N, class A> DPB_D vec_t<T, N> repack(const Values<A, N> &in)
{
    vec_t<T, N> v;
    if constexpr (is_half_v<T> && N % 2 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 2)
            *reinterpret_cast<__half2 *>(v.v + i) = __float22half2_rn(in.p[i / 2]);
    }
    else {
#pragma unroll
        for (int i = 0; i < N; ++i) v.v[i] = from_acc<T>(in.get(i));
    }
    return v;
}

// N elements at p (aligned to the accesses, which are of at most 16 bytes), through the read-only path:
// for arrays that the kernel does not write.
template <class A, int N, class W> DPB_D void load_values(const W *p, Values<A, N> &out)
{
    constexpr int part = N * sizeof(W) > 16 ? 16 / static_cast<int>(sizeof(W)) : N;
#pragma unroll
    for (int k = 0; k < N; k += part) {
        Values<A, part> some;
        unpack<A, part, W>(load_vec<vec_t<W, part>>(p + k), some);
#pragma unroll
        for (int j = 0; j < part; ++j) out.set(k + j, some.get(j));
    }
}

// 16 bytes of elements from an address that is aligned to its elements only: the two aligned accesses around it,
// shifted into place (about 15 instructions, against one load an element), where both lie in the array [lo, hi).
template <class T, int VEC> DPB_D vec_t<T, VEC> load_anywhere(const T *p, const T *lo, const T *hi)
{
    using V = vec_t<T, VEC>;
    static_assert(sizeof(V) == 16, "whole accesses");
    const int off = static_cast<int>(reinterpret_cast<uintptr_t>(p) & 15);
    if (off == 0) return load_vec<V>(p);
    const T *q = reinterpret_cast<const T *>(reinterpret_cast<uintptr_t>(p) - off);
    V out;
    if (q >= lo && q + 2 * VEC <= hi) {
        const int4 a = __ldg(reinterpret_cast<const int4 *>(q)), b = __ldg(reinterpret_cast<const int4 *>(q) + 1);
        uint32_t w[8] = {uint32_t(a.x), uint32_t(a.y), uint32_t(a.z), uint32_t(a.w),
                         uint32_t(b.x), uint32_t(b.y), uint32_t(b.z), uint32_t(b.w)};
#pragma unroll
        for (int i = 0; i < 6; ++i) w[i] = off & 8 ? w[i + 2] : w[i];
        if constexpr (sizeof(T) <= 4) {
#pragma unroll
            for (int i = 0; i < 5; ++i) w[i] = off & 4 ? w[i + 1] : w[i];
        }
        if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], (off & 2) * 8);
        }
        int4 r = make_int4(int(w[0]), int(w[1]), int(w[2]), int(w[3]));
        out = *reinterpret_cast<V *>(&r);
    }
    else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) out.v[j] = p[j];
    }
    return out;
}

// ------------------------------------------------------------------- rows fetched ahead into shared memory
// Copy of one access (16, 8 or 4 bytes) into shared memory that does not wait (2 bytes: a plain copy).
template <class V> DPB_D void copy_async(V *shared, const V *global)
{
    if constexpr (sizeof(V) == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(shared))),
                     "l"(global)
                     : "memory");
    else if constexpr (sizeof(V) >= 4)
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(shared))),
                     "l"(global), "n"(sizeof(V))
                     : "memory");
    else *shared = *global;
}
DPB_D void copy_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> DPB_D void copy_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <class T> struct Span {
    const T *lo, *hi;   // an array's elements
};

// The accesses of one thread to a row of n elements: ITEMS accesses of VEC elements, `width` threads apart.
// Where a row starts `mis` elements behind a 16-byte boundary the accesses start at that boundary (the
// columns are shifted by mis), so that every access is aligned; the first and the last then reach into
// the neighbouring rows, which is read (and not used) where it lies inside the array, and go element by
// element at the array's ends.  SHIFT = false: every row is aligned and n is a multiple of VEC.
template <class T, int VEC, int ITEMS, bool SHIFT> struct RowAccess {
    using V = vec_t<T, VEC>;
    int t, width, n, mis;
    DPB_D int column(int i) const { return (i * width + t) * VEC - (SHIFT ? mis : 0); }
    DPB_D bool any(int i) const { return column(i) < n && (!SHIFT || column(i) > -VEC); }
    DPB_D bool whole(int i) const { return !SHIFT || (column(i) >= 0 && column(i) + VEC <= n); }
    DPB_D bool has(int i, int j) const { return column(i) + j >= 0 && column(i) + j < n; }
    // zeros in the slots that no fetch will fill, for `rows` rows of the ring
    DPB_D void clear(V *slot, int stride, int rows) const
    {
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            if (any(i)) continue;
            V v;
#pragma unroll
            for (int j = 0; j < VEC; ++j) v.v[j] = from_acc<T>(acc_t<T>(0));
            for (int k = 0; k < rows; ++k) slot[(k * ITEMS + i) * stride] = v;
        }
    }
    // into the thread's own slots of shared memory, `stride` accesses apart; [lo, hi): the array
    DPB_D void fetch(const T *row, V *slot, int stride, const T *lo, const T *hi) const
    {
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            if (!any(i)) continue;
            const T *p = row + column(i);
            if (whole(i) || (p >= lo && p + VEC <= hi)) copy_async(slot + i * stride, reinterpret_cast<const V *>(p));
            else {
                V v;
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    if (has(i, j)) v.v[j] = p[j];
                slot[i * stride] = v;
            }
        }
    }
    // zeros in place of what is not in the row
    template <class A> DPB_D void clip(int i, Values<A, VEC> &v) const
    {
        if (whole(i)) return;
#pragma unroll
        for (int j = 0; j < VEC; ++j)
            if (!has(i, j)) v.set(j, A(0));
    }
    // `aligned`: this row lies on the boundaries that the columns were shifted for
    DPB_D void store(T *row, int i, const V &v, bool aligned) const
    {
        T *p = row + column(i);
        if (whole(i) && (!SHIFT || aligned)) {
            *reinterpret_cast<V *>(p) = v;
            return;
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j)
            if (has(i, j)) p[j] = v.v[j];
    }
    // values of an array of n elements that goes with the columns (a weight); `otherwise` outside
    template <class A, class W> DPB_D void load(const W *w, int i, Values<A, VEC> &out, A otherwise) const
    {
        out.fill(otherwise);
        if (!w || !any(i)) return;
        if constexpr (!SHIFT) load_values<A, VEC, W>(w + column(i), out);
        else {
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                if (has(i, j)) out.set(j, to_acc<A>(w[column(i) + j]));
        }
    }
};

// Elements between the 16-byte boundary below p and p.
template <class T> DPB_D int misalignment(const T *p)
{
    return static_cast<int>(reinterpret_cast<uintptr_t>(p) % 16) / static_cast<int>(sizeof(T));
}

}  // namespace dpb
