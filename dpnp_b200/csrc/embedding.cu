// Embedding lookup and its gradient.
//
//   out[i] = scale * table[id_i]            (a row of zeros where id_i is outside [0, V))
//   dtable[v] = scale * sum_{i : id_i = v} dout[i]
//
// The gradient is a sum of rows by key.  It is taken over the tokens sorted by id, so that every row
// of the table is written exactly once, by one owner, in an order that does not depend on timing:
//   1. a stable radix sort of (id, position), which also marks the ids that occur;
//   2. one launch that sums the runs of equal ids, a chunk of 32 to 128 sorted tokens a block (whole runs go to the table,
//      the parts of runs that cross a chunk's border to a workspace, so that a frequent id does not wait for
//      one block), and writes zeros to the rows that do not occur;
//   3. the sums of the parts, in order.
// Sums are float (double for float64 data), in ascending order of the positions within a chunk and of
// the chunks; the scale multiplies the finished sum, and the result is rounded once.
#include "row_ops.cuh"

namespace dpb {

constexpr int kThreads = 256;
constexpr int kAccesses = 4;   // of a thread, kThreads apart: in flight together

// The accesses of all rows in one sequence: access e of a matrix with `per_row` accesses a row.  A block
// takes kThreads * kAccesses consecutive ones, so that narrow rows share a block and wide ones are split.
struct RowSequence {
    FastDiv32 per_row;
    DPB_D void start(int64_t first, int64_t &row, uint32_t &rest) const
    {
        if (first < (int64_t(1) << 31)) {
            uint32_t q;
            per_row.divmod(static_cast<uint32_t>(first), q, rest);
            row = q;
        }
        else {
            row = first / per_row.d;
            rest = static_cast<uint32_t>(first - row * per_row.d);
        }
    }
};

// Rows shared out to groups of 2^bits threads of a block, as many as a row has accesses (rounded up to a power of two,
// at most the block): no division at all, for the stores of zeros.
constexpr int kRows = 4;   // of a thread

struct RowGroups {
    int bits;
    DPB_HD int width() const { return 1 << bits; }
    DPB_HD int groups() const { return kThreads >> bits; }
    DPB_D uint32_t lane() const { return threadIdx.x & (width() - 1); }
    DPB_D uint32_t group() const { return threadIdx.x >> bits; }
};

// Access k of a row that starts `mis` elements behind a 16-byte boundary begins at column k VEC - mis: all but the
// first and the last are whole and aligned.  A row of n elements has at most n + VEC - 1 over VEC of them (rounded up).
template <class T, int VEC> struct ShiftedColumn {
    int64_t c;
    int64_t n;
    DPB_D ShiftedColumn(const T *row, uint32_t k, int64_t n_) : c(int64_t(k) * VEC - misalignment_of(row)), n(n_) {}
    static DPB_D int misalignment_of(const T *row)
    {
        return static_cast<int>(reinterpret_cast<uintptr_t>(row) % (VEC * sizeof(T))) / static_cast<int>(sizeof(T));
    }
    DPB_D bool whole() const { return c >= 0 && c + VEC <= n; }
    DPB_D bool has(int j) const { return c + j >= 0 && c + j < n; }
    // from a row that may start anywhere; zeros outside it
    template <class S> DPB_D vec_t<S, VEC> load(const S *row, const Span<S> &array) const
    {
        if (whole()) {
            if constexpr (VEC * sizeof(S) == 16) return load_anywhere<S, VEC>(row + c, array.lo, array.hi);
        }
        vec_t<S, VEC> v;
#pragma unroll
        for (int j = 0; j < VEC; ++j) v.v[j] = has(j) ? row[c + j] : from_acc<S>(acc_t<S>(0));
        return v;
    }
    DPB_D void store(T *row, const vec_t<T, VEC> &v) const
    {
        if (whole()) *reinterpret_cast<vec_t<T, VEC> *>(row + c) = v;
        else
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                if (has(j)) row[c + j] = v.v[j];
    }
};

// ----------------------------------------------------------------------------------------- forward
// A copy with a gather: bound by memory, so four accesses in flight a thread.  SHIFT: rows start anywhere; the stores
// are aligned, the loads shifted into place.
template <class T, class I, bool SHIFT>
__global__ void __launch_bounds__(kThreads) embedding_kernel(const T *table, int64_t ld, Span<T> array, const I *ids, acc_t<T> scale,
                                                             T *out, RowMap om, int64_t vocab, int64_t tokens, int64_t n,
                                                             RowSequence seq)
{
    using A = acc_t<T>;
    constexpr int VEC = vec_width<T>();
    using V = vec_t<T, VEC>;
    cudaGridDependencySynchronize();
    int64_t row;
    uint32_t rest;
    seq.start(int64_t(blockIdx.x) * (kThreads * kAccesses), row, rest);
    int64_t token[kAccesses], id[kAccesses];
    uint32_t c[kAccesses];
#pragma unroll
    for (int k = 0; k < kAccesses; ++k) {
        uint32_t q;
        seq.per_row.divmod(rest + k * kThreads + threadIdx.x, q, c[k]);
        token[k] = row + q;
        id[k] = token[k] < tokens ? static_cast<int64_t>(ids[token[k]]) : -1;
    }
    V v[kAccesses];
#pragma unroll
    for (int k = 0; k < kAccesses; ++k) {
        if (id[k] < 0 || id[k] >= vocab) continue;
        const T *from = table + id[k] * ld;
        if constexpr (SHIFT)
            v[k] = ShiftedColumn<T, VEC>(out + om(static_cast<uint32_t>(token[k])), c[k], n).load(from, array);
        else v[k] = load_vec<V>(from + int64_t(c[k]) * VEC);
    }
#pragma unroll
    for (int k = 0; k < kAccesses; ++k) {
        if (token[k] >= tokens) continue;
        Values<A, VEC> u;
        u.fill(0);
        if (id[k] >= 0 && id[k] < vocab) {
            unpack<A, VEC, T>(v[k], u);
            u.mul(scale);
        }
        T *to = out + om(static_cast<uint32_t>(token[k]));
        const V w = repack<T, VEC, A>(u);
        if constexpr (SHIFT) ShiftedColumn<T, VEC>(to, c[k], n).store(to, w);
        else *reinterpret_cast<V *>(to + int64_t(c[k]) * VEC) = w;
    }
}

// ---------------------------------------------------------------------------------- sort of the ids
// Least significant digit first, `bits` of at most 9 bits a pass; the key of an id outside the table
// is `vocab`, which sorts behind all rows.  A tile of kTile tokens belongs to one block, a contiguous
// part of it to each warp, so that ranks within a digit follow the positions (a stable sort).
// hist[tile][digit] holds the tiles' counts; every placing block forms its own first places from them (up
// to kJoinedTiles tiles: one launch a pass, the next pass's counts by integer atomics on the way, whose
// order does not matter), or a scan kernel does that for all.
constexpr int kTile = 2048;
constexpr int kSortThreads = kThreads;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kMaxDigits = 512;
constexpr int kJoinedTiles = 64;

// Zeros for some rows of a matrix: the sort occupies few SMs, and its launches carry blocks that begin with the
// gradient's zeros (of rows that occur, too: they are written again later).
struct ZeroRows {
    char *base;
    int64_t row_bytes;     // from one row to the next
    int64_t bytes;         // of a row
    int item;              // bytes of an element
    RowGroups groups;      // accesses of 16 bytes, shifted to the rows' starts
    int64_t rows, first;   // first row of this launch
    int64_t blocks;
    DPB_HD int64_t block_rows() const { return int64_t(groups.groups()) * kRows; }
};
// `skip` (or null): rows that are written by others
DPB_D void zero_rows(const ZeroRows &z, int64_t block, const uint8_t *skip)
{
    const int64_t row0 = z.first + block * z.block_rows() + z.groups.group();
    bool mine[kRows];
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
        const int64_t row = row0 + k * z.groups.groups();
        mine[k] = row < z.rows && !(skip && skip[row]);
    }
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
        if (!mine[k]) continue;
        char *start = z.base + (row0 + k * z.groups.groups()) * z.row_bytes;
        const int64_t mis = static_cast<int64_t>(reinterpret_cast<uintptr_t>(start) % 16);
        for (int64_t at = int64_t(z.groups.lane()) * 16 - mis; at < z.bytes; at += int64_t(z.groups.width()) * 16) {
            if (at >= 0 && at + 16 <= z.bytes) *reinterpret_cast<int4 *>(start + at) = make_int4(0, 0, 0, 0);
            else
                for (int64_t i = max(at, int64_t(0)); i < min(at + 16, z.bytes); i += z.item) {
                    if (z.item == 2) *reinterpret_cast<short *>(start + i) = 0;
                    else if (z.item == 4) *reinterpret_cast<int *>(start + i) = 0;
                    else *reinterpret_cast<long long *>(start + i) = 0;
                }
        }
    }
}

struct SortIn {
    const void *ids;      // of type I in the first pass
    const uint32_t *key;  // sorted by the earlier digits in the later ones
    const uint32_t *pos;
};

constexpr int kRounds = kTile / kSortThreads;   // items a thread, 32 apart in its warp's part of the tile

struct SortItems {
    uint32_t key[kRounds], pos[kRounds];
    uint32_t valid;   // bit k: item k exists
};

// All items of a thread at once: the loads do not wait for one another.
template <class I> DPB_D void load_items(const SortIn &in, bool first, int64_t n, int64_t vocab, SortItems &it)
{
    const int64_t begin = int64_t(blockIdx.x) * kTile + (threadIdx.x >> 5) * (kTile / kSortWarps) + (threadIdx.x & 31);
    it.valid = 0;
#pragma unroll
    for (int k = 0; k < kRounds; ++k) {
        const int64_t i = begin + k * 32;
        it.key[k] = it.pos[k] = 0;
        if (i >= n) continue;
        it.valid |= 1u << k;
        if (first) {
            const int64_t id = static_cast<int64_t>(static_cast<const I *>(in.ids)[i]);
            it.key[k] = static_cast<uint32_t>(id >= 0 && id < vocab ? id : vocab);
            it.pos[k] = static_cast<uint32_t>(i);
        }
        else {
            it.key[k] = in.key[i];
            it.pos[k] = in.pos[i];
        }
    }
}

// Counts of a warp's part of the tile per digit.  Lanes with the same digit elect their lowest lane.
DPB_D void warp_count(const SortItems &it, int shift, uint32_t mask, uint32_t *count)
{
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int k = 0; k < kRounds; ++k) {
        const bool valid = it.valid >> k & 1;
        const uint32_t digit = valid ? (it.key[k] >> shift) & mask : ~0u;
        const unsigned same = __match_any_sync(0xffffffffu, digit);
        if (valid && lane == __ffs(same) - 1) count[digit] += __popc(same);
        __syncwarp();
    }
}

// Calls put(k, place) for the items in order: places of a digit from count[digit] on, which advances.
template <class F> DPB_D void warp_place(const SortItems &it, int shift, uint32_t mask, uint32_t *count, F put)
{
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int k = 0; k < kRounds; ++k) {
        const bool valid = it.valid >> k & 1;
        const uint32_t digit = valid ? (it.key[k] >> shift) & mask : ~0u;
        const unsigned same = __match_any_sync(0xffffffffu, digit);
        if (valid) put(k, count[digit] + __popc(same & ((1u << lane) - 1)));
        __syncwarp();
        if (valid && lane == __ffs(same) - 1) count[digit] += __popc(same);
        __syncwarp();
    }
}

DPB_D void clear_counts(uint32_t (&count)[kSortWarps][kMaxDigits])
{
    for (int d = threadIdx.x; d < kSortWarps * kMaxDigits; d += kSortThreads) (&count[0][0])[d] = 0;
}

// Counts of one digit; `later` counters behind them (of the later passes' tiles) are set to zero, and the marks
// of the ids too (`marks` of 4 ids, or none).
template <class I>
__global__ void __launch_bounds__(kSortThreads) sort_count_kernel(SortIn in, bool first, int64_t n, int64_t vocab, int shift,
                                                                  int bits, uint32_t *hist, int tiles, int later, uint32_t *mark, int64_t marks,
                                                                  ZeroRows zero)
{
    __shared__ uint32_t count[kSortWarps][kMaxDigits];
    cudaGridDependencySynchronize();
    if (blockIdx.x >= tiles) return zero_rows(zero, blockIdx.x - tiles, nullptr);
    SortItems it;
    load_items<I>(in, first, n, vocab, it);
    const int digits = 1 << bits;
    clear_counts(count);
    for (int d = threadIdx.x; d < later * digits; d += kSortThreads)
        hist[(int64_t(1 + d / digits) * tiles + blockIdx.x) * digits + d % digits] = 0;
    for (int64_t i = int64_t(blockIdx.x) * kSortThreads + threadIdx.x; i < marks; i += int64_t(tiles) * kSortThreads) mark[i] = 0;
    __syncthreads();
    warp_count(it, shift, digits - 1, count[threadIdx.x >> 5]);
    __syncthreads();
    for (int d = threadIdx.x; d < digits; d += kSortThreads) {
        uint32_t s = 0;
        for (int w = 0; w < kSortWarps; ++w) s += count[w][d];
        hist[int64_t(blockIdx.x) * digits + d] = s;
    }
}

// First place of every (tile, digit) in place of its count, by one block: the digits' totals are scanned,
// then each digit runs through its tiles.
__global__ void __launch_bounds__(kMaxDigits) sort_scan_kernel(uint32_t *hist, int64_t tiles, int digits)
{
    __shared__ uint32_t total[kMaxDigits];
    cudaGridDependencySynchronize();
    const int d = threadIdx.x;
    uint32_t s = 0;
    if (d < digits)
        for (int64_t t = 0; t < tiles; ++t) s += hist[t * digits + d];
    total[d] = s;
    __syncthreads();
    if (d == 0) {
        uint32_t at = 0;
        for (int k = 0; k < digits; ++k) {
            const uint32_t c = total[k];
            total[k] = at;
            at += c;
        }
    }
    __syncthreads();
    if (d >= digits) return;
    uint32_t at = total[d];
    for (int64_t t = 0; t < tiles; ++t) {
        const uint32_t c = hist[t * digits + d];
        hist[t * digits + d] = at;
        at += c;
    }
}

// Exclusive scan of kMaxDigits counters in shared memory by kSortThreads threads, two counters each.
DPB_D void scan_digits(uint32_t *v, uint32_t *warp_sum)
{
    static_assert(kMaxDigits == 2 * kSortThreads, "two counters a thread");
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t a = v[2 * threadIdx.x], b = v[2 * threadIdx.x + 1];
    uint32_t s = a + b;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const uint32_t t = __shfl_up_sync(0xffffffffu, s, d);
        if (lane >= d) s += t;
    }
    if (lane == 31) warp_sum[warp] = s;
    __syncthreads();
    uint32_t before = s - a - b;
    for (int w = 0; w < warp; ++w) before += warp_sum[w];
    v[2 * threadIdx.x] = before;
    v[2 * threadIdx.x + 1] = before + a;
    __syncthreads();
}

// Turns the warps' counts of each digit into the warps' first places, from the digit's first place on.
DPB_D void warp_places(uint32_t (&count)[kSortWarps][kMaxDigits], int d, uint32_t from)
{
    for (int w = 0; w < kSortWarps; ++w) {
        const uint32_t c = count[w][d];
        count[w][d] = from;
        from += c;
    }
}

// Moves every (key, position) to its place: first place of its digit and tile, plus the earlier warps' counts
// of the digit, plus its rank in its own warp's part.  JOINED: `hist` holds counts; `next` (or null) gathers
// the counts of the next digit in the tiles that the items move to.  The last pass (mark not null) marks the ids.
template <class I, bool JOINED>
__global__ void __launch_bounds__(kSortThreads) sort_place_kernel(SortIn in, bool first, int64_t n, int64_t vocab, int shift,
                                                                  int bits, const uint32_t *hist, uint32_t *next,
                                                                  uint32_t *key_out, uint32_t *pos_out, uint8_t *mark, int tiles,
                                                                  ZeroRows zero)
{
    __shared__ uint32_t count[kSortWarps][kMaxDigits];
    __shared__ uint32_t place[kMaxDigits], warp_sum[kSortWarps];
    cudaGridDependencySynchronize();
    if (blockIdx.x >= tiles) return zero_rows(zero, blockIdx.x - tiles, nullptr);
    SortItems it;
    load_items<I>(in, first, n, vocab, it);
    const int digits = 1 << bits, d0 = 2 * threadIdx.x;
    clear_counts(count);
    uint2 earlier = {0, 0}, all = {0, 0};   // this thread's two digits: in the tiles before, in all tiles
    if (d0 < digits) {
        const uint2 *h = reinterpret_cast<const uint2 *>(hist + d0);
        if constexpr (JOINED) {
#pragma unroll 16
            for (int t = 0; t < tiles; ++t) {
                const uint2 c = h[t * digits / 2];
                if (t < static_cast<int>(blockIdx.x)) {
                    earlier.x += c.x;
                    earlier.y += c.y;
                }
                all.x += c.x;
                all.y += c.y;
            }
        }
        else earlier = h[int64_t(blockIdx.x) * digits / 2];
    }
    place[d0] = all.x;
    place[d0 + 1] = all.y;
    __syncthreads();
    if constexpr (JOINED) scan_digits(place, warp_sum);
    const uint32_t mask = digits - 1;
    uint32_t *mine = count[threadIdx.x >> 5];
    warp_count(it, shift, mask, mine);
    __syncthreads();
    if (d0 < digits) {
        warp_places(count, d0, place[d0] + earlier.x);
        warp_places(count, d0 + 1, place[d0 + 1] + earlier.y);
    }
    __syncthreads();
    warp_place(it, shift, mask, mine, [&](int k, uint32_t to) {
        key_out[to] = it.key[k];
        pos_out[to] = it.pos[k];
        if (JOINED && next) atomicAdd(next + (to / kTile) * digits + ((it.key[k] >> (shift + bits)) & mask), 1u);
        if (mark && it.key[k] < vocab) mark[it.key[k]] = 1;
    });
}

// All passes of up to kTile tokens by one block, through shared memory.
template <class I>
__global__ void __launch_bounds__(kSortThreads) sort_tile_kernel(const I *ids, int64_t n, int64_t vocab, int passes, int bits,
                                                                 uint32_t *key_out, uint32_t *pos_out, uint8_t *mark, int64_t marks,
                                                                 ZeroRows zero)
{
    __shared__ uint32_t count[kSortWarps][kMaxDigits];
    __shared__ uint32_t place[kMaxDigits], warp_sum[kSortWarps], keys[kTile], positions[kTile];
    cudaGridDependencySynchronize();
    if (blockIdx.x >= 1) return zero_rows(zero, blockIdx.x - 1, nullptr);
    SortItems it;
    load_items<I>({ids, nullptr, nullptr}, true, n, vocab, it);
    for (int64_t i = threadIdx.x; i < marks; i += kSortThreads) reinterpret_cast<uint32_t *>(mark)[i] = 0;
    const int d0 = 2 * threadIdx.x;
    const uint32_t mask = (1u << bits) - 1;
    uint32_t *mine = count[threadIdx.x >> 5];
    for (int p = 0; p < passes; ++p) {
        if (p > 0) {
            const int begin = (threadIdx.x >> 5) * (kTile / kSortWarps) + (threadIdx.x & 31);
#pragma unroll
            for (int k = 0; k < kRounds; ++k) {
                if (!(it.valid >> k & 1)) continue;
                it.key[k] = keys[begin + k * 32];
                it.pos[k] = positions[begin + k * 32];
            }
        }
        clear_counts(count);
        __syncthreads();
        warp_count(it, p * bits, mask, mine);
        __syncthreads();
        for (int d = d0; d < d0 + 2; ++d) {
            uint32_t c = 0;
            for (int w = 0; w < kSortWarps; ++w) c += count[w][d];
            place[d] = c;
        }
        __syncthreads();
        scan_digits(place, warp_sum);
        warp_places(count, d0, place[d0]);
        warp_places(count, d0 + 1, place[d0 + 1]);
        __syncthreads();
        const bool last = p == passes - 1;
        warp_place(it, p * bits, mask, mine, [&](int k, uint32_t to) {
            (last ? key_out : keys)[to] = it.key[k];
            (last ? pos_out : positions)[to] = it.pos[k];
            if (last && it.key[k] < vocab) mark[it.key[k]] = 1;
        });
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------------------- gradient
constexpr int kMaxChunk = 128;  // sorted tokens of a block, at most
constexpr int kInFlight = 8;    // rows' loads of a thread in flight

// The first blocks sum runs: block (chunk k, column tile) walks its tokens in order.  A run that lies in the chunk goes
// to the table; part[2 k] takes the sum of one that came in from chunk k - 1 (and may go on), part[2 k + 1]
// of one that starts here and goes on.  The other blocks write the rows that do not occur.  Every `stride`-th block
// is one of the first kind: reads and writes overlap.
template <class T, class O, bool SHIFT>
__global__ void __launch_bounds__(kThreads) embedding_sums_kernel(const T *dout, RowMap dm, Span<T> array, const uint32_t *key,
                                                                  const uint32_t *pos, uint32_t tokens, const uint8_t *mark,
                                                                  acc_t<T> *part, acc_t<T> scale, O *dtable, int64_t ld,
                                                                  uint32_t vocab, int64_t n, uint32_t per_row, uint32_t sum_blocks,
                                                                  FastDiv32 tiles, FastDiv32 stride, ZeroRows zero, uint32_t chunk)
{
    using A = acc_t<T>;
    constexpr int VEC = vec_width<T>(), flight = SHIFT ? kInFlight / 2 : kInFlight;
    using V = vec_t<T, VEC>;
    using VO = vec_t<O, VEC>;
    using Vals = Values<A, VEC>;
    const auto write = [&](int64_t v, uint32_t c, const Vals &s) {
        const VO w = repack<O, VEC, A>(s);
        O *to = dtable + v * ld;
        if constexpr (SHIFT) ShiftedColumn<O, VEC>(to, c, n).store(to, w);
        else *reinterpret_cast<VO *>(to + int64_t(c) * VEC) = w;
    };
    cudaGridDependencySynchronize();
    uint32_t block, off;
    stride.divmod(blockIdx.x, block, off);
    if (off != 0 || block >= sum_blocks) return zero_rows(zero, blockIdx.x - min(block + (off != 0), sum_blocks), mark);
    __shared__ uint32_t keys[kMaxChunk + 2];   // with the token before and the token behind the chunk
    __shared__ int64_t rows[kMaxChunk];
    uint32_t k, tile;
    tiles.divmod(block, k, tile);
    const uint32_t begin = k * chunk, count = min(tokens - begin, chunk);
    if (threadIdx.x < count + 2) {
        const int64_t i = int64_t(begin) + threadIdx.x - 1;
        keys[threadIdx.x] = i >= 0 && i < tokens ? key[i] : ~0u;
    }
    if (threadIdx.x < count) rows[threadIdx.x] = dm(pos[begin + threadIdx.x]);
    __syncthreads();
    const uint32_t c = tile * kThreads + threadIdx.x;
    if (c >= per_row) return;
    Vals s, u;
    s.fill(0);
    bool whole = keys[0] != keys[1];   // the current run starts in this chunk
    for (uint32_t i0 = 0; i0 < count; i0 += flight) {
        V v[flight];
#pragma unroll
        for (int j = 0; j < flight; ++j) {
            if (i0 + j >= count || keys[i0 + j + 1] >= vocab) continue;
            const T *from = dout + rows[i0 + j];
            if constexpr (SHIFT) v[j] = ShiftedColumn<O, VEC>(dtable + int64_t(keys[i0 + j + 1]) * ld, c, n).load(from, array);
            else v[j] = load_vec<V>(from + int64_t(c) * VEC);
        }
#pragma unroll
        for (int j = 0; j < flight; ++j) {
            const uint32_t i = i0 + j;
            if (i >= count) break;
            const uint32_t id = keys[i + 1];
            if (id >= vocab) return;   // behind all rows of the table
            unpack<A, VEC, T>(v[j], u);
            s.add(u);
            const bool ends = keys[i + 2] != id;
            if (!ends && i + 1 < count) continue;
            if (whole && ends) {
                s.mul(scale);
                write(id, c, s);
            }
            else *reinterpret_cast<Vals *>(part + (int64_t(2 * k + whole) * per_row + c) * VEC) = s;
            s.fill(0);
            whole = true;
        }
    }
}

// Runs over several chunks: the block of the chunk in which one ends adds its parts in order.
template <class A, class O, int VEC, bool SHIFT>
__global__ void __launch_bounds__(kThreads) embedding_join_kernel(const uint32_t *key, uint32_t tokens, const A *part, A scale,
                                                                  O *dtable, int64_t ld, uint32_t vocab, int64_t n,
                                                                  uint32_t per_row, FastDiv32 tiles, uint32_t chunk)
{
    using Vals = Values<A, VEC>;
    cudaGridDependencySynchronize();
    uint32_t before, tile;
    tiles.divmod(blockIdx.x, before, tile);
    const uint32_t k = before + 1, begin = k * chunk, end = min(tokens, begin + chunk);
    const uint32_t id = key[begin];
    // a run that came in and ends here
    if (id >= vocab || key[begin - 1] != id || (end < tokens && key[end - 1] == id && key[end] == id)) return;
    const uint32_t c = tile * kThreads + threadIdx.x;
    // chunks before this one whose last token belongs to the run, a warp at a time
    uint32_t first = k;   // the first chunk that the run came into
    for (;;) {
        const int64_t at = int64_t(first) - 1 - (threadIdx.x & 31);   // chunk `at` passes the run on to at + 1
        const unsigned on = __ballot_sync(0xffffffffu, at >= 1 && key[at * chunk - 1] == id);
        const int run = on == 0xffffffffu ? 32 : __ffs(~on) - 1;
        first -= run;
        if (run < 32) break;
    }
    if (c >= per_row) return;
    const Vals *p = reinterpret_cast<const Vals *>(part) + c;
    Vals s = p[int64_t(2 * (first - 1) + 1) * per_row];
#pragma unroll 8
    for (uint32_t g = first; g <= k; ++g) s.add(p[int64_t(2 * g) * per_row]);
    s.mul(scale);
    const vec_t<O, VEC> w = repack<O, VEC, A>(s);
    O *to = dtable + id * ld;
    if constexpr (SHIFT) ShiftedColumn<O, VEC>(to, c, n).store(to, w);
    else *reinterpret_cast<vec_t<O, VEC> *>(to + int64_t(c) * VEC) = w;
}

// --------------------------------------------------------------------------------------- launchers
struct EmbedArgs {
    const dpb_array *table, *ids, *out;
    RowMap om;
    int64_t tokens, vocab, n, ld;
    double scale;
};

// Accesses of 16 bytes a row: without and with a shift to the row's start (two partial ones then).
static int64_t row_accesses(int64_t n, int vec, bool shift)
{
    return shift ? ceil_div(n + vec - 1, vec) : n / vec;
}

template <class T> static Span<T> span_of(const dpb_array &a)
{
    const void *lo, *hi;
    array_bounds(a, lo, hi);
    return {static_cast<const T *>(lo), static_cast<const T *>(hi)};
}

static RowGroups row_groups(int64_t per_row)
{
    RowGroups g = {0};
    while (g.width() < kThreads && g.width() < per_row) ++g.bits;
    return g;
}

static unsigned sequence_blocks(int64_t rows, int64_t per_row)
{
    return static_cast<unsigned>(ceil_div(rows * per_row, kThreads * kAccesses));
}

template <class T, class I, bool SHIFT> static void launch_forward(const EmbedArgs &a, cudaStream_t s)
{
    const int64_t per_row = row_accesses(a.n, vec_width<T>(), SHIFT);
    launch_after_previous(embedding_kernel<T, I, SHIFT>, sequence_blocks(a.tokens, per_row), unsigned(kThreads), s,
                          static_cast<const T *>(a.table->data), a.ld, span_of<T>(*a.table), static_cast<const I *>(a.ids->data),
                          acc_t<T>(a.scale), static_cast<T *>(a.out->data), a.om, a.vocab, a.tokens, a.n,
                          RowSequence{FastDiv32(uint32_t(per_row))});
}

template <class T, class I> static int run_forward(const EmbedArgs &a, cudaStream_t s)
{
    constexpr int wide = vec_width<T>();
    const RowMap table = {0, a.ld, FastDiv32(1)};
    const bool aligned = row_vector(a.out->data, a.om, a.n, sizeof(T), wide) == wide &&
                         row_vector(a.table->data, table, a.n, sizeof(T), wide) == wide;
    if (aligned) launch_forward<T, I, false>(a, s);
    else launch_forward<T, I, true>(a, s);
    note_kernel("embedding");
    return check_launch("embedding");
}

static int64_t sort_words(int64_t n)   // of the sort's workspace
{
    return 4 * n + 4 * ceil_div(n, kTile) * kMaxDigits;
}

// Zeros that a launch of the sort writes on the side: what the memory takes in the 5 (counting) and 10 (placing)
// us that the sort's own blocks need.
constexpr int64_t kZerosCounting = int64_t(32) << 20, kZerosPlacing = int64_t(64) << 20;

// Moves `zero` on to the next launch's share, of `bytes` at most; its number of blocks.
static int64_t take_zeros(ZeroRows &z, int64_t bytes)
{
    z.first = std::min(z.rows, z.first + z.blocks * z.block_rows());
    const int64_t rows = std::min(z.rows - z.first, bytes / z.bytes);
    z.blocks = rows == z.rows - z.first ? ceil_div(rows, z.block_rows()) : rows / z.block_rows();
    return z.blocks;
}

// Sorted keys and positions of the ids in `work` (two pairs of arrays of `n`, then the counters of the passes), and
// marks of the ids that occur.
template <class I> static void sort_ids(const void *ids, int64_t n, int64_t vocab, uint32_t *work, uint8_t *mark, uint32_t *&key,
                                        uint32_t *&pos, ZeroRows &zero, cudaStream_t s)
{
    int bits = 1;
    while ((int64_t(1) << bits) <= vocab) ++bits;
    const int passes = (bits + 8) / 9, width = (bits + passes - 1) / passes;
    const int64_t tiles = std::max<int64_t>(1, ceil_div(n, kTile)), counters = tiles << width, marks = ceil_div(vocab, 4);
    const unsigned block = kSortThreads;
    const auto grid = [&](int64_t bytes) { return static_cast<unsigned>(tiles + take_zeros(zero, bytes)); };
    if (tiles == 1) {
        key = work;
        pos = work + n;
        const unsigned blocks = grid(kZerosPlacing);
        launch_after_previous(sort_tile_kernel<I>, blocks, block, s, static_cast<const I *>(ids), n, vocab, passes, width, key, pos, mark,
                              marks, zero);
        note_kernel("sort_tile");
        return;
    }
    const bool joined = tiles <= kJoinedTiles;
    uint32_t *bufs[2][2] = {{work, work + n}, {work + 2 * n, work + 3 * n}};
    uint32_t *hist = work + 4 * n;
    SortIn in = {ids, nullptr, nullptr};
    for (int p = 0; p < passes; ++p) {
        const int shift = p * width;
        key = bufs[p & 1][0];
        pos = bufs[p & 1][1];
        uint8_t *last = p + 1 == passes ? mark : nullptr;
        if (!joined || p == 0) {
            const unsigned blocks = grid(kZerosCounting);
            launch_after_previous(sort_count_kernel<I>, blocks, block, s, in, p == 0, n, vocab, shift, width, hist, int(tiles),
                                  joined ? passes - 1 : 0, reinterpret_cast<uint32_t *>(mark), p == 0 ? marks : 0, zero);
            note_kernel("sort_count");
        }
        if (joined) {
            uint32_t *next = p + 1 < passes ? hist + counters : nullptr;
            const unsigned blocks = grid(kZerosPlacing);
            launch_after_previous(sort_place_kernel<I, true>, blocks, block, s, in, p == 0, n, vocab, shift, width, hist, next, key, pos,
                                  last, int(tiles), zero);
            hist += counters;
        }
        else {
            launch_after_previous(sort_scan_kernel, 1u, unsigned(kMaxDigits), s, hist, tiles, 1 << width);
            note_kernel("sort_scan");
            const unsigned blocks = grid(kZerosPlacing);
            launch_after_previous(sort_place_kernel<I, false>, blocks, block, s, in, p == 0, n, vocab, shift, width, hist,
                                  static_cast<uint32_t *>(nullptr), key, pos, last, int(tiles), zero);
        }
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

template <class T, class O, bool SHIFT>
static void run_sums(const EmbedGradArgs &a, void *work, size_t head, uint32_t chunk, cudaStream_t s)
{
    using A = acc_t<T>;
    constexpr int VEC = vec_width<T>();
    uint32_t *w = static_cast<uint32_t *>(work), *key = nullptr, *pos = nullptr;
    uint8_t *mark = reinterpret_cast<uint8_t *>(w + sort_words(a.tokens));
    A *part = reinterpret_cast<A *>(static_cast<char *>(work) + head);
    const int64_t per_row = row_accesses(a.n, VEC, SHIFT), tiles = ceil_div(per_row, kThreads), chunks = ceil_div(a.tokens, int64_t(chunk));
    O *dtable = static_cast<O *>(a.dtable->data);
    ZeroRows zero = {reinterpret_cast<char *>(dtable), a.ld * int64_t(sizeof(O)), a.n * int64_t(sizeof(O)), int(sizeof(O)),
                     row_groups(row_accesses(a.n, 16 / int(sizeof(O)), SHIFT || a.n * sizeof(O) % 16 != 0)), a.vocab, 0, 0};
    if (a.ids->typenum == DPB_INT32) sort_ids<int32_t>(a.ids->data, a.tokens, a.vocab, w, mark, key, pos, zero, s);
    else sort_ids<int64_t>(a.ids->data, a.tokens, a.vocab, w, mark, key, pos, zero, s);
    const int64_t sums = chunks * tiles, zeros = take_zeros(zero, INT64_MAX);
    if (sums + zeros > 0) {
        const int64_t stride = sums > 0 ? std::max<int64_t>(1, (sums + zeros) / sums) : 1;
        launch_after_previous(embedding_sums_kernel<T, O, SHIFT>, static_cast<unsigned>(sums + zeros), unsigned(kThreads), s,
                              static_cast<const T *>(a.dout->data), a.dm, a.tokens > 0 ? span_of<T>(*a.dout) : Span<T>{nullptr, nullptr},
                              static_cast<const uint32_t *>(key), static_cast<const uint32_t *>(pos), uint32_t(a.tokens),
                              static_cast<const uint8_t *>(mark), part, A(a.scale), dtable, a.ld, uint32_t(a.vocab), a.n,
                              uint32_t(per_row), uint32_t(sums), FastDiv32(uint32_t(tiles)), FastDiv32(uint32_t(stride)), zero, chunk);
        note_kernel("embedding_sums");
    }
    if (chunks < 2) return;
    launch_after_previous(embedding_join_kernel<A, O, VEC, SHIFT>, static_cast<unsigned>((chunks - 1) * tiles), unsigned(kThreads), s,
                          static_cast<const uint32_t *>(key), uint32_t(a.tokens), static_cast<const A *>(part), A(a.scale), dtable, a.ld,
                          uint32_t(a.vocab), a.n, uint32_t(per_row), FastDiv32(uint32_t(tiles)), chunk);
    note_kernel("embedding_join");
}

template <class T, class O> static int run_backward(const EmbedGradArgs &a, cudaStream_t s)
{
    using A = acc_t<T>;
    constexpr int wide = vec_width<T>();
    const RowMap table = {0, a.ld, FastDiv32(1)};
    const bool shift = (a.tokens > 0 && row_vector(a.dout->data, a.dm, a.n, sizeof(T), wide) != wide) ||
                       row_vector(a.dtable->data, table, a.n, sizeof(O), wide) != wide;
    const int64_t per_row = row_accesses(a.n, wide, shift);
    // long chunks leave fewer parts of frequent ids to add up, short ones give few tokens enough blocks
    const int64_t tiles = ceil_div(per_row, kThreads);
    uint32_t chunk = 32;
    while (chunk < kMaxChunk && a.tokens / (2 * chunk) * tiles >= 4 * device_props().sm_count) chunk *= 2;
    // sorted keys and positions, counters, a mark a row; parts of runs
    const size_t words = static_cast<size_t>(sort_words(a.tokens) + ceil_div(a.vocab, 4)) * 4;
    const size_t head = (words + 255) / 256 * 256;
    void *work = nullptr;
    DPB_TRY(dpb_malloc(head + static_cast<size_t>(2 * ceil_div(a.tokens, int64_t(chunk)) * per_row * wide) * sizeof(A), s, &work));
    if (shift) run_sums<T, O, true>(a, work, head, chunk, s);
    else run_sums<T, O, false>(a, work, head, chunk, s);
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
    if (n > kMaxRows / 2) return set_error(DPB_ERR_VALUE, "%s: rows of more than 2^30 - 1 elements are not supported", what);
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
