// Embedding lookup and its gradient.
//
//   out[i] = scale * table[id_i]            (a row of zeros where id_i is outside [0, V))
//   dtable[v] = scale * sum_{i : id_i = v} dout[i]
//
// The gradient is a sum of rows by key.  It is taken over the tokens sorted by id, so that every row
// of the table is written exactly once, by one owner, in an order that does not depend on timing:
//   1. a stable radix sort of (id, position);
//   2. the first sorted index of every id (binary search);
//   3. runs of one id that cross a multiple of kChunk sorted tokens are summed per chunk, so that a
//      frequent id does not wait for one block;
//   4. every table row is the sum of its tokens' rows, of its chunks' sums, or zero.
// Sums are float (double for float64 data), in ascending order of the positions within a chunk and of
// the chunks; the scale multiplies the finished sum, and the result is rounded once.
#include "row_ops.cuh"

namespace dpb {

constexpr int kThreads = 256;

// ----------------------------------------------------------------------------------------- forward
template <class T, class I>
__global__ void __launch_bounds__(kThreads) embedding_kernel(const T *table, int64_t ld, const I *ids, acc_t<T> scale, T *out,
                                                             RowMap om, int64_t vocab, int64_t n)
{
    using A = acc_t<T>;
    const uint32_t r = blockIdx.x;
    const int64_t id = static_cast<int64_t>(ids[r]);
    T *o = out + om(r);
    const bool known = id >= 0 && id < vocab;
    const T *row = table + (known ? id * ld : 0);
    for (int64_t c = threadIdx.x; c < n; c += kThreads)
        o[c] = known ? from_acc<T>(to_acc<A>(row[c]) * scale) : from_acc<T>(A(0));
}

// ---------------------------------------------------------------------------------- sort of the ids
// Least significant digit first, `bits` of at most 9 bits a pass; the key of an id outside the table
// is `vocab`, which sorts behind all rows.  A tile of kTile tokens belongs to one block, a contiguous
// part of it to each warp, so that ranks within a digit follow the positions (a stable sort).
constexpr int kTile = 4096;
constexpr int kSortThreads = 256;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kMaxDigits = 512;

struct SortIn {
    const void *ids;      // of type I in the first pass
    const uint32_t *key;  // sorted by the earlier digits in the later ones
    const uint32_t *pos;
};

template <class I> DPB_D void sort_item(const SortIn &in, bool first, int64_t i, int64_t vocab, uint32_t &key, uint32_t &pos)
{
    if (first) {
        const int64_t id = static_cast<int64_t>(static_cast<const I *>(in.ids)[i]);
        key = static_cast<uint32_t>(id >= 0 && id < vocab ? id : vocab);
        pos = static_cast<uint32_t>(i);
    }
    else {
        key = in.key[i];
        pos = in.pos[i];
    }
}

// Counts of a warp's part of the tile per digit.  Lanes with the same digit elect their lowest lane.
template <class I>
DPB_D void warp_count(const SortIn &in, bool first, int64_t begin, int64_t end, int64_t vocab, int shift, uint32_t mask,
                      uint32_t *count)
{
    const int lane = threadIdx.x & 31;
    for (int64_t at = begin; at < end; at += 32) {
        const int64_t i = at + lane;
        uint32_t key = 0, pos, digit = ~0u;
        if (i < end) {
            sort_item<I>(in, first, i, vocab, key, pos);
            digit = (key >> shift) & mask;
        }
        const unsigned same = __match_any_sync(0xffffffffu, digit);
        if (i < end && lane == __ffs(same) - 1) count[digit] += __popc(same);
        __syncwarp();
    }
}

// hist[digit][tile]
template <class I>
__global__ void __launch_bounds__(kSortThreads) sort_count_kernel(SortIn in, bool first, int64_t n, int64_t vocab, int shift,
                                                                  int bits, uint32_t *hist)
{
    __shared__ uint32_t count[kSortWarps][kMaxDigits];
    const int digits = 1 << bits, warp = threadIdx.x >> 5;
    for (int d = threadIdx.x; d < kSortWarps * kMaxDigits; d += kSortThreads) (&count[0][0])[d] = 0;
    __syncthreads();
    constexpr int part = kTile / kSortWarps;
    const int64_t begin = min(n, int64_t(blockIdx.x) * kTile + int64_t(warp) * part), end = min(n, begin + part);
    warp_count<I>(in, first, begin, end, vocab, shift, digits - 1, count[warp]);
    __syncthreads();
    for (int d = threadIdx.x; d < digits; d += kSortThreads) {
        uint32_t s = 0;
        for (int w = 0; w < kSortWarps; ++w) s += count[w][d];
        hist[int64_t(d) * gridDim.x + blockIdx.x] = s;
    }
}

// Exclusive scan of `n` counters in place by one block.
__global__ void __launch_bounds__(1024) sort_scan_kernel(uint32_t *hist, int64_t n)
{
    __shared__ uint32_t warp_sum[32];
    __shared__ uint32_t carry_s;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) carry_s = 0;
    __syncthreads();
    for (int64_t base = 0; base < n; base += 1024) {
        const int64_t i = base + threadIdx.x;
        const uint32_t v = i < n ? hist[i] : 0;
        uint32_t s = v;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const uint32_t t = __shfl_up_sync(0xffffffffu, s, d);
            if (lane >= d) s += t;
        }
        if (lane == 31) warp_sum[warp] = s;
        __syncthreads();
        if (warp == 0) {
            uint32_t t = warp_sum[lane];
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const uint32_t u = __shfl_up_sync(0xffffffffu, t, d);
                if (lane >= d) t += u;
            }
            warp_sum[lane] = t;
        }
        __syncthreads();
        const uint32_t before = carry_s + (warp > 0 ? warp_sum[warp - 1] : 0);
        if (i < n) hist[i] = before + s - v;
        __syncthreads();
        if (threadIdx.x == 0) carry_s += warp_sum[31];
        __syncthreads();
    }
}

// Moves every (key, position) to its place: first place of its digit and tile (from the scan), plus the
// earlier warps' counts of the digit, plus its rank in its own warp's part.
template <class I>
__global__ void __launch_bounds__(kSortThreads) sort_place_kernel(SortIn in, bool first, int64_t n, int64_t vocab, int shift,
                                                                  int bits, const uint32_t *hist, uint32_t *key_out,
                                                                  uint32_t *pos_out)
{
    __shared__ uint32_t count[kSortWarps][kMaxDigits];
    const int digits = 1 << bits, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int d = threadIdx.x; d < kSortWarps * kMaxDigits; d += kSortThreads) (&count[0][0])[d] = 0;
    __syncthreads();
    constexpr int part = kTile / kSortWarps;
    const int64_t begin = min(n, int64_t(blockIdx.x) * kTile + int64_t(warp) * part), end = min(n, begin + part);
    const uint32_t mask = digits - 1;
    warp_count<I>(in, first, begin, end, vocab, shift, mask, count[warp]);
    __syncthreads();
    for (int d = threadIdx.x; d < digits; d += kSortThreads) {
        uint32_t s = hist[int64_t(d) * gridDim.x + blockIdx.x];
        for (int w = 0; w < kSortWarps; ++w) {
            const uint32_t c = count[w][d];
            count[w][d] = s;
            s += c;
        }
    }
    __syncthreads();
    for (int64_t at = begin; at < end; at += 32) {
        const int64_t i = at + lane;
        uint32_t key = 0, pos = 0, digit = ~0u;
        if (i < end) {
            sort_item<I>(in, first, i, vocab, key, pos);
            digit = (key >> shift) & mask;
        }
        const unsigned same = __match_any_sync(0xffffffffu, digit);
        if (i < end) {
            const uint32_t to = count[warp][digit] + __popc(same & ((1u << lane) - 1));
            key_out[to] = key;
            pos_out[to] = pos;
        }
        __syncwarp();
        if (i < end && lane == __ffs(same) - 1) count[warp][digit] += __popc(same);
        __syncwarp();
    }
}

// ---------------------------------------------------------------------------------------- gradient
constexpr int kChunk = 128;

// first[v] = number of sorted keys below v, for v = 0 .. vocab
__global__ void __launch_bounds__(kThreads) segment_start_kernel(const uint32_t *key, int64_t n, int64_t vocab, uint32_t *first)
{
    const int64_t v = int64_t(blockIdx.x) * kThreads + threadIdx.x;
    if (v > vocab) return;
    int64_t lo = 0, hi = n;
    while (lo < hi) {
        const int64_t mid = (lo + hi) >> 1;
        if (key[mid] < static_cast<uint32_t>(v)) lo = mid + 1;
        else hi = mid;
    }
    first[v] = static_cast<uint32_t>(lo);
}

// Sums of the runs that cross a chunk's borders: part[2 k] for a run that came in from chunk k - 1,
// part[2 k + 1] for one that starts in chunk k and goes on in chunk k + 1.
template <class T>
__global__ void __launch_bounds__(kThreads) embedding_chunk_kernel(const T *dout, RowMap dm, const uint32_t *key,
                                                                   const uint32_t *pos, const uint32_t *first,
                                                                   int64_t n_tokens, int64_t vocab, int64_t n, acc_t<T> *part)
{
    using A = acc_t<T>;
    const int64_t k = blockIdx.x, begin = k * kChunk, end = min(n_tokens, begin + kChunk);
    for (int side = 0; side < 2; ++side) {
        const uint32_t id = key[side == 0 ? begin : end - 1];
        if (id >= vocab) continue;
        const int64_t from = first[id], to = first[id + 1];
        if (side == 0 ? from >= begin : (to <= end || from < begin)) continue;
        const int64_t b = max(begin, from), e = min(end, to);
        for (int64_t c = int64_t(blockIdx.y) * kThreads + threadIdx.x; c < n; c += int64_t(gridDim.y) * kThreads) {
            A s = 0;
            for (int64_t i = b; i < e; ++i) s += to_acc<A>(dout[dm(pos[i]) + c]);
            part[(2 * k + side) * n + c] = s;
        }
    }
}

template <class T, class O>
__global__ void __launch_bounds__(kThreads) embedding_rows_kernel(const T *dout, RowMap dm, const uint32_t *pos,
                                                                  const uint32_t *first, const acc_t<T> *part, acc_t<T> scale,
                                                                  int64_t n, O *dtable, int64_t ld)
{
    using A = acc_t<T>;
    const int64_t v = blockIdx.x;
    const int64_t from = first[v], to = first[v + 1];
    O *o = dtable + v * ld;
    const int64_t k0 = from / kChunk, k1 = (to - 1) / kChunk;
    for (int64_t c = threadIdx.x; c < n; c += kThreads) {
        A s = 0;
        if (to > from) {
            if (k0 == k1)
                for (int64_t i = from; i < to; ++i) s += to_acc<A>(dout[dm(pos[i]) + c]);
            else {
                s = part[(2 * k0 + 1) * n + c];
                for (int64_t k = k0 + 1; k <= k1; ++k) s += part[2 * k * n + c];
            }
        }
        o[c] = from_acc<O>(s * scale);
    }
}

// --------------------------------------------------------------------------------------- launchers
struct EmbedArgs {
    const dpb_array *table, *ids, *out;
    RowMap om;
    int64_t tokens, vocab, n, ld;
    double scale;
};

template <class T, class I> static int run_forward(const EmbedArgs &a, cudaStream_t s)
{
    embedding_kernel<T, I><<<static_cast<unsigned>(a.tokens), kThreads, 0, s>>>(
        static_cast<const T *>(a.table->data), a.ld, static_cast<const I *>(a.ids->data), acc_t<T>(a.scale),
        static_cast<T *>(a.out->data), a.om, a.vocab, a.n);
    note_kernel("embedding");
    return check_launch("embedding");
}

// Sorted keys and positions of the ids in `work` (4 arrays of `n`, then the counters).
template <class I> static void sort_ids(const void *ids, int64_t n, int64_t vocab, uint32_t *work, uint32_t *&key, uint32_t *&pos,
                                        cudaStream_t s)
{
    int bits = 1;
    while ((int64_t(1) << bits) <= vocab) ++bits;
    const int passes = (bits + 8) / 9, width = (bits + passes - 1) / passes;
    const int64_t tiles = ceil_div(n, kTile);
    uint32_t *bufs[2][2] = {{work, work + n}, {work + 2 * n, work + 3 * n}};
    uint32_t *hist = work + 4 * n;
    SortIn in = {ids, nullptr, nullptr};
    for (int p = 0; p < passes; ++p) {
        const int shift = p * width;
        const unsigned grid = static_cast<unsigned>(tiles);
        sort_count_kernel<I><<<grid, kSortThreads, 0, s>>>(in, p == 0, n, vocab, shift, width, hist);
        note_kernel("sort_count");
        sort_scan_kernel<<<1, 1024, 0, s>>>(hist, tiles << width);
        note_kernel("sort_scan");
        key = bufs[p & 1][0];
        pos = bufs[p & 1][1];
        sort_place_kernel<I><<<grid, kSortThreads, 0, s>>>(in, p == 0, n, vocab, shift, width, hist, key, pos);
        note_kernel("sort_place");
        in = {nullptr, key, pos};
    }
}

struct EmbedGradArgs {
    const dpb_array *dout, *ids, *dtable;
    RowMap dm;
    int64_t tokens, vocab, n, ld;
    double scale;
};

template <class T, class O> static int run_backward(const EmbedGradArgs &a, cudaStream_t s)
{
    using A = acc_t<T>;
    const int64_t tiles = ceil_div(a.tokens, kTile), chunks = ceil_div(a.tokens, kChunk);
    const size_t words = static_cast<size_t>(4 * a.tokens + tiles * kMaxDigits + a.vocab + 1);
    const size_t head = (words * 4 + 255) / 256 * 256;
    void *work = nullptr;
    DPB_TRY(dpb_malloc(head + static_cast<size_t>(2 * chunks * a.n) * sizeof(A), s, &work));
    uint32_t *w = static_cast<uint32_t *>(work), *key = nullptr, *pos = nullptr;
    uint32_t *first = w + 4 * a.tokens + tiles * kMaxDigits;
    A *part = reinterpret_cast<A *>(static_cast<char *>(work) + head);
    if (a.tokens > 0) {
        if (a.ids->typenum == DPB_INT32) sort_ids<int32_t>(a.ids->data, a.tokens, a.vocab, w, key, pos, s);
        else sort_ids<int64_t>(a.ids->data, a.tokens, a.vocab, w, key, pos, s);
    }
    segment_start_kernel<<<static_cast<unsigned>(ceil_div(a.vocab + 1, kThreads)), kThreads, 0, s>>>(key, a.tokens, a.vocab, first);
    note_kernel("segment_start");
    const T *dout = static_cast<const T *>(a.dout->data);
    if (a.tokens > kChunk) {
        const dim3 grid(static_cast<unsigned>(chunks), static_cast<unsigned>(std::min<int64_t>(ceil_div(a.n, kThreads), 16)));
        embedding_chunk_kernel<T><<<grid, kThreads, 0, s>>>(dout, a.dm, key, pos, first, a.tokens, a.vocab, a.n, part);
        note_kernel("embedding_chunk");
    }
    embedding_rows_kernel<T, O><<<static_cast<unsigned>(a.vocab), kThreads, 0, s>>>(
        dout, a.dm, pos, first, part, A(a.scale), a.n, static_cast<O *>(a.dtable->data), a.ld);
    note_kernel("embedding_rows");
    const int st = check_launch("embedding_backward");
    dpb_free(work, s);
    return st;
}

// The table (or its gradient): two dimensions, rows of unit stride.
static int check_table(const dpb_array &t, int64_t &vocab, int64_t &n, int64_t &ld, const char *what)
{
    if (t.nd != 2) return set_error(DPB_ERR_VALUE, "%s: a two-dimensional array is needed", what);
    DPB_TRY(check_float_type(t, what));
    vocab = t.shape[0];
    n = t.shape[1];
    if (vocab > kMaxRows) return set_error(DPB_ERR_VALUE, "%s: more than 2^31 - 1 rows are not supported", what);
    const std::vector<int64_t> st = strides_of(t);
    if (n > 1 && st[1] != 1) return set_error(DPB_ERR_VALUE, "%s: rows of unit stride are needed", what);
    ld = st[0];
    return DPB_OK;
}

static int check_ids(const dpb_array &ids, int64_t &tokens)
{
    if (ids.typenum != DPB_INT32 && ids.typenum != DPB_INT64)
        return set_error(DPB_ERR_TYPE, "ids: int32 or int64 is needed, got %s", type_name(ids.typenum));
    DPB_TRY(check_c_contiguous(ids, "ids"));
    tokens = num_elements(ids);
    if (tokens > kMaxRows) return set_error(DPB_ERR_VALUE, "more than 2^31 - 1 ids are not supported");
    return DPB_OK;
}

}  // namespace dpb

using namespace dpb;

extern "C" {

int dpb_embedding(const dpb_array *table, const dpb_array *ids, double scale, const dpb_array *out, void *stream)
{
    DPB_TRY(check_operand(table, "table"));
    DPB_TRY(check_operand(ids, "ids"));
    DPB_TRY(check_operand(out, "out"));
    EmbedArgs a = {};
    DPB_TRY(check_table(*table, a.vocab, a.n, a.ld, "table"));
    DPB_TRY(check_ids(*ids, a.tokens));
    DPB_TRY(check_same_device(*table, *ids));
    DPB_TRY(check_same_device(*table, *out));
    DPB_TRY(check_type(*out, table->typenum, "out"));
    DPB_TRY(check_shape(*out, ids->shape, ids->nd, a.n, "out"));
    DPB_TRY(check_output(*out, "out"));
    if (a.tokens == 0 || a.n == 0) return DPB_OK;
    DPB_TRY(check_row_map(*out, a.om, "out"));
    DPB_TRY(check_no_overlaps({table, ids}, {out}));
    a.table = table, a.ids = ids, a.out = out, a.scale = scale;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool narrow = ids->typenum == DPB_INT32;
    switch (table->typenum) {
    case DPB_HALF: return narrow ? run_forward<half_t, int32_t>(a, s) : run_forward<half_t, int64_t>(a, s);
    case DPB_FLOAT: return narrow ? run_forward<float, int32_t>(a, s) : run_forward<float, int64_t>(a, s);
    default: return narrow ? run_forward<double, int32_t>(a, s) : run_forward<double, int64_t>(a, s);
    }
}

int dpb_embedding_backward(const dpb_array *dout, const dpb_array *ids, double scale, const dpb_array *dtable, void *stream)
{
    DPB_TRY(check_operand(dout, "dout"));
    DPB_TRY(check_operand(ids, "ids"));
    DPB_TRY(check_operand(dtable, "dtable"));
    EmbedGradArgs a = {};
    DPB_TRY(check_table(*dtable, a.vocab, a.n, a.ld, "dtable"));
    DPB_TRY(check_ids(*ids, a.tokens));
    DPB_TRY(check_same_device(*dtable, *ids));
    DPB_TRY(check_same_device(*dtable, *dout));
    DPB_TRY(check_float_type(*dout, "dout"));
    if (dtable->typenum != dout->typenum && !(dout->typenum == DPB_HALF && dtable->typenum == DPB_FLOAT))
        return set_error(DPB_ERR_TYPE, "dtable: type %s does not go with %s data", type_name(dtable->typenum),
                         type_name(dout->typenum));
    DPB_TRY(check_shape(*dout, ids->shape, ids->nd, a.n, "dout"));
    DPB_TRY(check_output(*dtable, "dtable"));
    if (a.vocab == 0 || a.n == 0) return DPB_OK;
    if (a.tokens > 0) DPB_TRY(check_row_map(*dout, a.dm, "dout"));
    DPB_TRY(check_no_overlaps({dout, ids}, {dtable}));
    a.dout = dout, a.ids = ids, a.dtable = dtable, a.scale = scale;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dout->typenum == DPB_DOUBLE) return run_backward<double, double>(a, s);
    if (dout->typenum == DPB_FLOAT) return run_backward<float, float>(a, s);
    return dtable->typenum == DPB_FLOAT ? run_backward<half_t, float>(a, s) : run_backward<half_t, half_t>(a, s);
}

}  // extern "C"
