// Host-side build of how the row operators walk the rows of an array (dpnp_b200/csrc/row_ops.cuh), so that the
// addresses the kernels take can be compared with the array's strides on a machine without a GPU.
// Built by tests/test_row_walk_host.py with nvcc; host code only, no kernel, no device call.
#include "../../dpnp_b200/csrc/row_ops.cuh"

#include "../../dpnp_b200/csrc/iterspace.cpp"

int dpb::set_error(int status, const char *, ...) { return status; }

using namespace dpb;

extern "C" {

// Element offsets of the rows r, r + step, ... below `rows`, as a group of threads comes by them.  Returns their
// number, -1 for rows that the kernels do not take.
long rw_walk(int nd, const int64_t *shape, const int64_t *strides, uint32_t r, uint32_t step, int64_t *offsets)
{
    const dpb_array a = {nullptr, nd, DPB_FLOAT, 0, 0, shape, strides};
    RowMap map;
    if (!make_row_map(a, map)) return -1;
    static const char origin[1] = {};
    const int64_t rows = count_rows(a);
    long n = 0;
    for (RowWalk<const char> walk(origin, map, r, step); r < rows; ++n) {
        offsets[n] = reinterpret_cast<intptr_t>(walk.p) - reinterpret_cast<intptr_t>(origin);
        r += step;
        if (r < rows) walk.next(r);
    }
    return n;
}

// Whether all rows are one and the same stride apart (-1 as above).
int rw_one_stride(int nd, const int64_t *shape, const int64_t *strides)
{
    const dpb_array a = {nullptr, nd, DPB_FLOAT, 0, 0, shape, strides};
    RowMap map;
    return make_row_map(a, map) ? map.one_stride() : -1;
}
}
