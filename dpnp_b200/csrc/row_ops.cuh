// Shared parts of the row operators (layer normalisation, embedding lookup, distillation loss):
// how the rows of a descriptor lie in memory, accumulation types, block-wide sums, and the argument
// checks of their entry points.
#pragma once

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
    DPB_D int64_t operator()(uint32_t r) const
    {
        uint32_t q, m;
        extent.divmod(r, q, m);
        return int64_t(q) * outer + int64_t(m) * inner;
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
    if (levels == 2) {
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

// -------------------------------------------------------------------------------- argument checks
constexpr int64_t kMaxRows = INT32_MAX;   // row numbers are divided with 31-bit arithmetic

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

// fmaf / fma under the library's -fmad=false
DPB_D float fma_(float a, float b, float c) { return fmaf(a, b, c); }
DPB_D double fma_(double a, double b, double c) { return fma(a, b, c); }
DPB_D float exp_(float a) { return expf(a); }
DPB_D double exp_(double a) { return exp(a); }
DPB_D float log_(float a) { return logf(a); }
DPB_D double log_(double a) { return log(a); }
DPB_D float sqrt_(float a) { return sqrtf(a); }
DPB_D double sqrt_(double a) { return sqrt(a); }

}  // namespace dpb
