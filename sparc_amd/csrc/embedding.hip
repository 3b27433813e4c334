// Lookup of scaled table rows by token, and the table's gradient by sorted tokens.
//
//     out[i, :] = round(scale * table[ids[i], :])
//     dT[v, :]  = round(scale * sum over i with ids[i] = v of g[i, :])         (rows without a token: 0)
//
// Gradient.  Four launches, no atomics on values, every sum in one fixed order:
//   tile_counts    a workgroup per tile of TILE tokens sorts their places by bucket (a bucket is 2^shift consecutive
//                  rows), stable, and writes where each bucket starts inside the tile;
//   bucket_rows    a workgroup per bucket walks its part of every tile in order and sorts it by row, stable: the places
//                  of every row in ascending order (`place`) and where each row's places end (`row_end`), a CSR matrix
//                  whose product with g is the gradient;
//   row_sums       the product.  Work is cut along the merged list of (places of row 0, row 0 done, places of row 1, ...)
//                  so that a worker has `per` items whatever the rows hold: long rows are cut, empty rows cost the
//                  store of their zeros and no separate fill.  A row of at most LONG_ROW places belongs to the worker
//                  that meets its first; a longer one leaves one partial sum per worker
//   join_rows      which are added in order (float64) here.  Usually nothing to do.
#include "elem.h"

namespace {

constexpr int TILE = 2048;         // tokens per workgroup of tile_counts
constexpr int MAX_BUCKETS = 2048;  // counters per wave of tile_counts
constexpr int WAVES = 4;
constexpr int BLOCK = 64 * WAVES;
constexpr int ROWS_AT_ONCE = 2048; // rows per pass of bucket_rows over its bucket
constexpr int LONG_ROW = 64;
constexpr int STAGE = 4096;        // items of a workgroup of row_sums at most
constexpr int AHEAD = 4;           // gradient rows in flight per worker
constexpr int JOIN_GRID = 256;

template <int DT>
struct Width {
    static constexpr int VE = 16 / sizeof(typename Elem<DT>::type);
};

// ---- lookup ------------------------------------------------------------------------------------------------

struct LookupArgs {
    const void* ids;
    const void* table;
    void* out;
    int64_t rows, ld, ldo, items;
    uint32_t per_row;      // vectors of an output row
    uint32_t dim;
    float scale;
    int wide_ids;
};

__device__ __forceinline__ int64_t token(const void* ids, const int wide, const int64_t i) {
    return wide ? static_cast<const int64_t*>(ids)[i] : static_cast<const int32_t*>(ids)[i];
}

// One 16-byte vector of an output row per thread and turn (an element of rows shorter than that).  A row's last vector
// ends with the row: it overlaps the one before it and both write the same values.
constexpr int TURNS = 4;           // vectors in flight per thread

template <int DT, int VE>
__global__ __launch_bounds__(BLOCK) void lookup_kernel(const LookupArgs a) {
    typedef typename Elem<DT>::type T;
    const T* table = static_cast<const T*>(a.table);
    T* out = static_cast<T*>(a.out);
    const int64_t step = static_cast<int64_t>(gridDim.x) * BLOCK;
    for (int64_t w0 = static_cast<int64_t>(blockIdx.x) * BLOCK + threadIdx.x; w0 < a.items; w0 += TURNS * step) {
        int64_t at[TURNS];
        Vec<DT, VE> v[TURNS];
        int64_t id[TURNS];
        int col[TURNS];
#pragma unroll
        for (int k = 0; k < TURNS; ++k) {
            const int64_t w = w0 + k * step;
            id[k] = -1;
            at[k] = -1;
            if (w < a.items) {
                const int64_t row = w / a.per_row;
                col[k] = min(static_cast<int>(w - row * a.per_row) * VE, static_cast<int>(a.dim) - VE);
                at[k] = row * a.ldo + col[k];
                id[k] = token(a.ids, a.wide_ids, row);
            }
        }
#pragma unroll
        for (int k = 0; k < TURNS; ++k)
            if (id[k] >= 0 && id[k] < a.rows) v[k].load(table + id[k] * a.ld + col[k]);
#pragma unroll
        for (int k = 0; k < TURNS; ++k) {
            if (at[k] < 0) continue;
            if (id[k] >= 0 && id[k] < a.rows) {
                if (a.scale != 1.f) {   // (a copy keeps the bits)
#pragma unroll
                    for (int i = 0; i < VE; ++i) v[k].set(i, v[k].get(i) * a.scale);
                }
            } else {
#pragma unroll
                for (int i = 0; i < VE; ++i) v[k].set(i, __builtin_nanf(""));
            }
            v[k].store(out + at[k]);
        }
    }
}

// ---- gradient ------------------------------------------------------------------------------------------------

// Everything the launches share.  tiles x buckets is bounded by n / TILE x MAX_BUCKETS: as large as the tokens.
struct GradArgs {
    const void* ids;
    const void* g;
    void* out;
    int64_t n, rows, ldg, padding;
    int64_t tiles, tile;       // number of tiles, tokens of a tile
    int64_t workers;
    int buckets, shift;
    int dim, wide_ids;
    int per;                   // items of a worker
    float scale;
    uint32_t* tile_start;      // [buckets + 1][tiles]: where a bucket starts inside a tile
    uint32_t* sorted;          // [n] places, by bucket inside a tile
    uint32_t* place;           // [n] places, by row
    uint32_t* row_end;         // [rows]
    uint32_t* long_rows;       // [1 + 3 * most]: count, then {row, first worker, last worker}
    float* part;               // [2 workers][dim]
};

// Lanes below this one whose key equals mine, among the lanes of `live`; *all: every such lane.
__device__ __forceinline__ int rank_among_equals(const uint32_t key, const int bits, const uint64_t live, uint64_t* all) {
    uint64_t same = live;
    for (int b = 0; b < bits; ++b) {
        const uint64_t ones = __ballot((key >> b) & 1u);
        same &= ((key >> b) & 1u) ? ones : ~ones;
    }
    *all = same;
    const uint64_t below = same & ((1ull << (threadIdx.x & 63)) - 1ull);
    return __popcll(below);
}

// Exclusive prefix sums over `count` x WAVES counters in LDS, key by key and inside a key wave by wave:
// cnt[w * count + k] becomes its start.  tot: WAVES words of LDS.  Returns the total.
__device__ uint32_t scan_counters(uint32_t* cnt, const int count, uint32_t* tot) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int each = (count + BLOCK - 1) / BLOCK;
    const int k0 = min(tid * each, count), k1 = min(k0 + each, count);
    uint32_t mine = 0;
    for (int k = k0; k < k1; ++k)
#pragma unroll
        for (int w = 0; w < WAVES; ++w) mine += cnt[w * count + k];
    uint32_t upto = mine;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const uint32_t other = __shfl_up(upto, off);
        if (lane >= off) upto += other;
    }
    if (lane == 63) tot[wave] = upto;
    __syncthreads();
    uint32_t base = upto - mine, total = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        if (w < wave) base += tot[w];
        total += tot[w];
    }
    for (int k = k0; k < k1; ++k)
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const uint32_t c = cnt[w * count + k];
            cnt[w * count + k] = base;
            base += c;
        }
    __syncthreads();
    return total;
}

__global__ __launch_bounds__(BLOCK) void tile_counts(const GradArgs a, const int bits) {
    extern __shared__ uint32_t cnt[];   // [WAVES][buckets]
    __shared__ uint32_t tot[WAVES];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t t = blockIdx.x, first = t * a.tile;
    const int64_t per_wave = a.tile / WAVES;
    const int64_t lo = min(first + wave * per_wave, a.n), hi = min(first + (wave + 1) * per_wave, a.n);
    uint32_t* mine = cnt + wave * a.buckets;
    if (t == 0 && threadIdx.x == 0) a.long_rows[0] = 0;
    for (int i = threadIdx.x; i < WAVES * a.buckets; i += BLOCK) cnt[i] = 0;
    __syncthreads();
    for (int64_t i = lo + lane; i < hi; i += 64) {
        const int64_t id = token(a.ids, a.wide_ids, i);
        if (id >= 0 && id < a.rows && id != a.padding) atomicAdd(mine + (id >> a.shift), 1u);
    }
    __syncthreads();
    const uint32_t total = scan_counters(cnt, a.buckets, tot);
    for (int b = threadIdx.x; b < a.buckets; b += BLOCK) a.tile_start[static_cast<int64_t>(b) * a.tiles + t] = cnt[b];
    if (threadIdx.x == 0) a.tile_start[static_cast<int64_t>(a.buckets) * a.tiles + t] = total;
    __syncthreads();   // (wave 0 moves its counters, which are the bucket starts, on)
    for (int64_t i0 = lo; i0 < hi; i0 += 64) {
        const int64_t i = i0 + lane;
        const int64_t id = i < hi ? token(a.ids, a.wide_ids, i) : -1;
        const bool ok = id >= 0 && id < a.rows && id != a.padding;
        const uint32_t b = ok ? static_cast<uint32_t>(id >> a.shift) : 0u;
        uint64_t same;
        const int r = rank_among_equals(b, bits, __ballot(ok), &same);
        if (ok) {
            const uint32_t at = mine[b];
            a.sorted[first + at + r] = static_cast<uint32_t>(i);
            if (r == 0) mine[b] = at + __popcll(same);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // the counters as the next turn's lanes find them
    }
}

// Element j of a bucket's part of the tiles: the tile whose running total covers it (run[t] = elements before tile t).
__device__ __forceinline__ int64_t tile_of(const uint32_t* run, const int tiles, const uint32_t j) {
    int lo = 0, hi = tiles;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (run[mid] <= j) lo = mid;
        else hi = mid;
    }
    return lo;
}

__global__ __launch_bounds__(BLOCK) void bucket_rows(const GradArgs a) {
    extern __shared__ uint32_t lds[];   // counters [WAVES][row_slots], run [tiles], where [tiles]
    __shared__ uint32_t tot[WAVES];
    __shared__ uint32_t before[WAVES];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t b = blockIdx.x;
    const int64_t row0 = b << a.shift;
    const int64_t in_bucket = min(static_cast<int64_t>(1) << a.shift, a.rows - row0);
    const int slots = static_cast<int>(min(in_bucket, static_cast<int64_t>(ROWS_AT_ONCE)));
    const int tiles = static_cast<int>(a.tiles);
    const int row_bits = min(a.shift, 11);               // (ROWS_AT_ONCE rows)
    uint32_t* cnt = lds;
    uint32_t* run = cnt + WAVES * min(1 << a.shift, ROWS_AT_ONCE);
    uint32_t* where = run + tiles;
    // the bucket's part of every tile: running totals, and the places before the bucket (its start in `place`)
    uint32_t start = 0, total = 0;
    for (int t0 = 0; t0 < tiles; t0 += BLOCK) {
        const int t = t0 + tid;
        uint32_t lo = 0, len = 0;
        if (t < tiles) {
            lo = a.tile_start[b * a.tiles + t];
            len = a.tile_start[(b + 1) * a.tiles + t] - lo;
            where[t] = lo;
        }
        uint32_t upto = len, low = lo;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const uint32_t other = __shfl_up(upto, off), o2 = __shfl_xor(low, off);
            if (lane >= off) upto += other;
            low += o2;
        }
        if (lane == 63) {
            tot[wave] = upto;
            before[wave] = low;
        }
        __syncthreads();
        uint32_t base = total;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            if (w < wave) base += tot[w];
            total += tot[w];
            start += before[w];
        }
        if (t < tiles) run[t] = base + upto - len;
        __syncthreads();
    }
    const uint32_t per_wave = ((total + BLOCK - 1) / BLOCK) * 64;
    const uint32_t lo = min(wave * per_wave, total), hi = min(lo + per_wave, total);
    uint32_t done = start;   // places of the passes before this one
    for (int64_t r0 = 0; r0 < in_bucket; r0 += slots) {
        const int count = static_cast<int>(min(in_bucket - r0, static_cast<int64_t>(slots)));
        for (int i = tid; i < WAVES * count; i += BLOCK) cnt[i] = 0;
        __syncthreads();
        uint32_t* mine = cnt + wave * count;
        for (int turn = 0; turn < 2; ++turn) {   // count, then place
            for (uint32_t j0 = lo; j0 < hi; j0 += 64) {
                const uint32_t j = j0 + lane;
                uint32_t i = 0, r = 0;
                bool ok = j < hi;
                if (ok) {
                    const int64_t t = tile_of(run, tiles, j);
                    i = a.sorted[t * a.tile + where[t] + (j - run[t])];
                    const int64_t local = token(a.ids, a.wide_ids, i) - row0 - r0;
                    ok = local >= 0 && local < count;
                    r = ok ? static_cast<uint32_t>(local) : 0u;
                }
                if (turn == 0) {
                    if (ok) atomicAdd(mine + r, 1u);
                } else {
                    uint64_t same;
                    const int k = rank_among_equals(r, row_bits, __ballot(ok), &same);
                    if (ok) {
                        const uint32_t at = mine[r];
                        a.place[done + at + k] = i;
                        if (k == 0) mine[r] = at + __popcll(same);
                    }
                    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                }
            }
            __syncthreads();
            if (turn == 0) {
                const uint32_t all = scan_counters(cnt, count, tot);
                // wave 0's counter of the next row is where this row ends
                for (int k = tid; k < count; k += BLOCK) a.row_end[row0 + r0 + k] = done + (k + 1 < count ? cnt[k + 1] : all);
                if (tid == 0) tot[0] = all;
                __syncthreads();
            }
        }
        done += tot[0];
        __syncthreads();
    }
}

// The point of the merged list with `diag` items before it: the smallest row r whose end item lies at or behind diag,
// i.e. row_end[r] + r >= diag; diag - r places lie before it.  (Items of row r: its places, then its end.)
__device__ __forceinline__ int64_t merge_row(const uint32_t* row_end, const int64_t rows, const int64_t diag) {
    // 64 probes at a time; the answer is in [lo, hi]
    int64_t lo = 0, hi = min(rows, diag);
    const int lane = threadIdx.x & 63;
    while (hi > lo) {
        const int64_t width = (hi - lo + 63) >> 6;
        const int64_t r = lo + lane * width;
        const bool below = r < hi && static_cast<int64_t>(row_end[r]) + r < diag;
        const int k = __popcll(__ballot(below));   // probes 0 .. k - 1 are below: the answer lies behind probe k - 1
        if (k == 0) return lo;
        const int64_t new_lo = lo + (k - 1) * width + 1;
        hi = min(hi, lo + k * width);
        lo = new_lo;
    }
    return lo;
}

// Workers are groups of `lanes` lanes (a power of two); lane u of a group owns VE columns of the slice blockIdx.y.
template <int DT, int VE>
__global__ __launch_bounds__(BLOCK) void row_sums(const GradArgs a, const int lanes_log2) {
    typedef typename Elem<DT>::type T;
    __shared__ uint32_t ends[STAGE + 2];                 // row_end of rows [row0 - 1, row1]
    __shared__ uint32_t places[STAGE + LONG_ROW];
    __shared__ int64_t edge[2];
    const T* g = static_cast<const T*>(a.g);
    T* out = static_cast<T*>(a.out);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int lanes = 1 << lanes_log2, in_group = BLOCK >> lanes_log2;
    const int u = tid & (lanes - 1);
    const int64_t first_worker = static_cast<int64_t>(blockIdx.x) * in_group;
    const int64_t all_places = a.rows > 0 ? a.row_end[a.rows - 1] : 0;
    const int64_t items = all_places + a.rows;
    const int64_t d0 = min(first_worker * a.per, items), d1 = min(d0 + static_cast<int64_t>(in_group) * a.per, items);
    if (d0 >= d1) return;                                // (the whole workgroup)
    if (wave < 2) {
        const int64_t r = merge_row(a.row_end, a.rows, wave ? d1 : d0);
        if (lane == 0) edge[wave] = r;
    }
    __syncthreads();
    const int64_t row0 = edge[0], row1 = edge[1];        // rows row0 .. row1 - 1 end in this workgroup's items
    const uint32_t e0 = static_cast<uint32_t>(d0 - row0), e1 = static_cast<uint32_t>(d1 - row1);
    const int n_ends = static_cast<int>(row1 - row0) + 2;   // ends[k] = row_end[row0 - 1 + k]
    for (int k = tid; k < n_ends; k += BLOCK) {
        const int64_t r = row0 - 1 + k;
        ends[k] = r < 0 ? 0u : r < a.rows ? a.row_end[r] : static_cast<uint32_t>(all_places);
    }
    const uint32_t e_last = min(e1 + LONG_ROW, static_cast<uint32_t>(all_places));
    for (uint32_t k = e0 + tid; k < e_last; k += BLOCK) places[k - e0] = a.place[k];
    __syncthreads();
    const int64_t worker = first_worker + (tid >> lanes_log2);
    const int64_t w0 = min(worker * a.per, items), w1 = min(w0 + a.per, items);
    const int col = min((blockIdx.y * lanes + u) * VE, a.dim - VE);
    if (w0 >= w1 || (static_cast<int>(blockIdx.y) * lanes + u) * VE >= a.dim) return;   // no barrier below
    // this worker's two points, as rows relative to row0
    auto split = [&](const int64_t d) {
        int lo = 0, hi = static_cast<int>(min(row1 - row0, d - d0));
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (static_cast<int64_t>(ends[mid + 1]) + row0 + mid < d) lo = mid + 1;
            else hi = mid;
        }
        return lo;
    };
    int r = split(w0), r_stop = split(w1);               // rows r .. r_stop - 1 end in [w0, w1)
    uint32_t e = static_cast<uint32_t>(w0 - row0 - r), e_stop = static_cast<uint32_t>(w1 - row0 - r_stop);
    bool inside = false;                                 // the first row began in an earlier worker
    if (e > ends[r]) {                                   // (ends[r]: where row r begins)
        if (ends[r + 1] - ends[r] <= LONG_ROW) {
            e = ends[r + 1];                             // an earlier worker has the whole row
            ++r;
        } else {
            inside = true;
        }
    }
    if (row0 + r_stop < a.rows && e_stop > ends[r_stop] && ends[r_stop + 1] - ends[r_stop] <= LONG_ROW) {
        e_stop = ends[r_stop + 1];                       // the row that is cut here is this worker's
        ++r_stop;
    }
    if (r > r_stop || (r == r_stop && e >= e_stop)) return;
    float acc[VE];
#pragma unroll
    for (int i = 0; i < VE; ++i) acc[i] = 0.f;
    auto finish_row = [&]() {
        if (inside) {
            float* p = a.part + (2 * worker) * a.dim + col;
#pragma unroll
            for (int i = 0; i < VE; ++i) p[i] = acc[i];
            if (u == 0 && blockIdx.y == 0) {             // the last piece of a long row: announce it
                const uint32_t k = atomicAdd(a.long_rows, 1u);
                a.long_rows[1 + 3 * k] = static_cast<uint32_t>(row0 + r);
                a.long_rows[2 + 3 * k] = static_cast<uint32_t>((row0 + r + ends[r]) / a.per);
                a.long_rows[3 + 3 * k] = static_cast<uint32_t>(worker);
            }
            inside = false;
        } else {
            Vec<DT, VE> v;
#pragma unroll
            for (int i = 0; i < VE; ++i) v.set(i, acc[i] * a.scale);
            v.store(out + (row0 + r) * a.dim + col);
        }
#pragma unroll
        for (int i = 0; i < VE; ++i) acc[i] = 0.f;
        ++r;
    };
    Vec<DT, VE> ahead[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
        if (e + k < e_stop) ahead[k].load(g + static_cast<int64_t>(places[e + k - e0]) * a.ldg + col);
    while (e < e_stop) {
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            if (e + k >= e_stop) break;
            while (ends[r + 1] <= e + k) finish_row();
#pragma unroll
            for (int i = 0; i < VE; ++i) acc[i] += ahead[k].get(i);
            if (e + k + AHEAD < e_stop) ahead[k].load(g + static_cast<int64_t>(places[e + k + AHEAD - e0]) * a.ldg + col);
        }
        e += AHEAD;
    }
    while (r < r_stop) finish_row();
    if (e_stop > ends[r_stop]) {                         // a long row goes on in the next worker
        float* p = a.part + (2 * worker + (inside ? 0 : 1)) * a.dim + col;
#pragma unroll
        for (int i = 0; i < VE; ++i) p[i] = acc[i];
    }
}

// Long rows: slice blockIdx.y of 64 columns, a lane per column; the waves take a quarter of the pieces each.
template <int DT>
__global__ __launch_bounds__(BLOCK) void join_rows(const GradArgs a) {
    typedef typename Elem<DT>::type T;
    __shared__ double sum[WAVES][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int col = blockIdx.y * 64 + lane;
    const uint32_t count = a.long_rows[0];
    for (uint32_t k = blockIdx.x; k < count; k += gridDim.x) {
        const int64_t row = a.long_rows[1 + 3 * k], first = a.long_rows[2 + 3 * k], last = a.long_rows[3 + 3 * k];
        const int64_t pieces = last - first + 1, each = (pieces + WAVES - 1) / WAVES;
        const int64_t lo = min(wave * each, pieces), hi = min(lo + each, pieces);
        double s = 0.0;
        if (col < a.dim)
            for (int64_t p = lo; p < hi; ++p)            // the first worker's piece begins the row: its second slot
                s += a.part[(2 * (first + p) + (p == 0 ? 1 : 0)) * a.dim + col];
        sum[wave][lane] = s;
        __syncthreads();
        if (wave == 0 && col < a.dim) {
            s = sum[0][lane];
#pragma unroll
            for (int w = 1; w < WAVES; ++w) s += sum[w][lane];
            static_cast<T*>(a.out)[row * a.dim + col] = Elem<DT>::down(static_cast<float>(s) * a.scale);
        }
        __syncthreads();
    }
}

// Sizes of the workspace's parts, from n, rows and dim alone.
struct Plan {
    int64_t tile, tiles, workers;
    int shift, buckets, per, lanes_log2, slices, in_group;
    size_t bytes;
};

int64_t ceil_div(const int64_t a, const int64_t b) { return (a + b - 1) / b; }

Plan plan_of(const int64_t n, const int64_t rows, const int dim, const int ve) {
    Plan p;
    p.tile = TILE * ceil_div(n > 0 ? n : 1, static_cast<int64_t>(TILE) * MAX_BUCKETS);   // at most MAX_BUCKETS tiles
    p.tiles = ceil_div(n, p.tile);
    p.shift = 0;
    while (ceil_div(rows, static_cast<int64_t>(1) << p.shift) > MAX_BUCKETS) ++p.shift;
    p.buckets = static_cast<int>(ceil_div(rows, static_cast<int64_t>(1) << p.shift));
    const int units = (dim + ve - 1) / ve;
    p.lanes_log2 = 0;
    while ((1 << p.lanes_log2) < units && p.lanes_log2 < 6) ++p.lanes_log2;
    p.slices = (units + (1 << p.lanes_log2) - 1) >> p.lanes_log2;
    p.in_group = BLOCK >> p.lanes_log2;
    // items of a worker: enough workers for every SIMD's wave slots first, up to 64 items then
    const int64_t wanted = ceil_div(n + rows, static_cast<int64_t>(8192) * 64 >> p.lanes_log2);
    p.per = static_cast<int>(wanted < 4 ? 4 : wanted > 64 ? 64 : wanted);
    if (static_cast<int64_t>(p.per) * p.in_group > STAGE) p.per = STAGE / p.in_group;
    p.workers = ceil_div(n + rows, p.per);
    return p;
}

template <typename F>
int launch_lookup(F&& f, const int dtype, const bool vectors) {
    if (dtype == SPARC_F32) return vectors ? f(lookup_kernel<SPARC_F32, 4>) : f(lookup_kernel<SPARC_F32, 1>);
    if (dtype == SPARC_BF16) return vectors ? f(lookup_kernel<SPARC_BF16, 8>) : f(lookup_kernel<SPARC_BF16, 1>);
    return vectors ? f(lookup_kernel<SPARC_F16, 8>) : f(lookup_kernel<SPARC_F16, 1>);
}

GradArgs carve(const Plan& p, const int64_t n, const int64_t rows, const int dim, void* ws, const size_t ws_bytes, bool* ok, size_t* used) {
    GradArgs a = {};
    WsCarver c(ws, ws_bytes);
    a.tile_start = c.take<uint32_t>(static_cast<size_t>(p.buckets + 1) * p.tiles);
    a.sorted = c.take<uint32_t>(n);
    a.place = c.take<uint32_t>(n);
    a.row_end = c.take<uint32_t>(rows);
    a.long_rows = c.take<uint32_t>(1 + 3 * (n / LONG_ROW + 1));
    a.part = c.take<float>(static_cast<size_t>(2) * p.workers * dim);
    *ok = c.ok();
    *used = c.off;
    return a;
}

int elements_of_16_bytes(const int dtype) { return dtype == SPARC_F32 ? 4 : 8; }

}  // namespace

extern "C" int sparc_embedding_fwd(int64_t n, int64_t rows, int64_t dim, int dtype, const void* ids, int ids_64, const void* table,
                                   int64_t ld, double scale, void* out, int64_t ldo, sparc_stream_t stream) {
    if (n < 0 || rows < 0 || dim < 0 || dtype < SPARC_F32 || dtype > SPARC_F16 || ld < dim || ldo < dim || !ids || !out || (rows > 0 && !table))
        return SPARC_ERR_ARG;
    if (n > SPARC_EMBEDDING_MAX || rows > SPARC_EMBEDDING_MAX || dim > SPARC_EMBEDDING_MAX_DIM) return SPARC_ERR_SIZE;
    if (n == 0 || dim == 0) return SPARC_OK;
    const int ve = elements_of_16_bytes(dtype);
    const bool vectors = dim >= ve;
    LookupArgs a;
    a.ids = ids;
    a.table = table;
    a.out = out;
    a.rows = rows;
    a.ld = ld;
    a.ldo = ldo;
    a.per_row = static_cast<uint32_t>(vectors ? (dim + ve - 1) / ve : dim);
    a.items = n * a.per_row;
    a.dim = static_cast<uint32_t>(dim);
    a.scale = static_cast<float>(scale);
    a.wide_ids = ids_64 ? 1 : 0;
    const int64_t blocks = ceil_div(a.items, static_cast<int64_t>(BLOCK) * TURNS);
    const unsigned grid = static_cast<unsigned>(blocks < (1 << 20) ? blocks : (1 << 20));
    return launch_lookup([&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(grid), dim3(BLOCK), 0, stream, a);
        SPARC_CHECK_LAUNCH();
        return SPARC_OK;
    }, dtype, vectors);
}

extern "C" size_t sparc_embedding_grad_workspace_bytes(int64_t n, int64_t rows, int64_t dim, int dtype) {
    if (n < 0 || rows < 0 || dim < 0 || n > SPARC_EMBEDDING_MAX || rows > SPARC_EMBEDDING_MAX || dim > SPARC_EMBEDDING_MAX_DIM ||
        dtype < SPARC_F32 || dtype > SPARC_F16)
        return 0;
    const int ve = elements_of_16_bytes(dtype);
    const Plan p = plan_of(n, rows, static_cast<int>(dim), dim >= ve ? ve : 1);
    bool ok;
    size_t used;
    carve(p, n, rows, static_cast<int>(dim), nullptr, 0, &ok, &used);
    return used;
}

namespace {

template <int DT, int VE>
int launch_grad(const GradArgs& a, const Plan& p, sparc_stream_t stream) {
    int bits = 0;
    while ((1 << bits) < p.buckets) ++bits;
    if (p.tiles > 0) {
        hipLaunchKernelGGL(tile_counts, dim3(static_cast<unsigned>(p.tiles)), dim3(BLOCK),
                           static_cast<size_t>(WAVES) * p.buckets * sizeof(uint32_t), stream, a, bits);
        SPARC_CHECK_LAUNCH();
    }
    const int64_t slots = (static_cast<int64_t>(1) << p.shift) < ROWS_AT_ONCE ? (1 << p.shift) : ROWS_AT_ONCE;
    hipLaunchKernelGGL(bucket_rows, dim3(static_cast<unsigned>(p.buckets)), dim3(BLOCK),
                       static_cast<size_t>(WAVES * slots + 2 * p.tiles) * sizeof(uint32_t), stream, a);
    SPARC_CHECK_LAUNCH();
    hipLaunchKernelGGL((row_sums<DT, VE>), dim3(static_cast<unsigned>(ceil_div(p.workers, p.in_group)), p.slices), dim3(BLOCK), 0, stream, a,
                       p.lanes_log2);
    SPARC_CHECK_LAUNCH();
    if (a.n > LONG_ROW) {
        hipLaunchKernelGGL((join_rows<DT>), dim3(JOIN_GRID, static_cast<unsigned>((a.dim + 63) / 64)), dim3(BLOCK), 0, stream, a);
        SPARC_CHECK_LAUNCH();
    }
    return SPARC_OK;
}

}  // namespace

extern "C" int sparc_embedding_grad(int64_t n, int64_t rows, int64_t dim, int dtype, const void* ids, int ids_64, const void* g,
                                    int64_t ldg, double scale, int64_t padding_idx, void* out, void* ws, size_t ws_bytes,
                                    sparc_stream_t stream) {
    if (n < 0 || rows < 0 || dim < 0 || dtype < SPARC_F32 || dtype > SPARC_F16 || ldg < dim || !out || !ws || (n > 0 && (!ids || !g)))
        return SPARC_ERR_ARG;
    if (n > SPARC_EMBEDDING_MAX || rows > SPARC_EMBEDDING_MAX || dim > SPARC_EMBEDDING_MAX_DIM) return SPARC_ERR_SIZE;
    if (rows == 0 || dim == 0) return SPARC_OK;
    const int ve = elements_of_16_bytes(dtype), used_ve = dim >= ve ? ve : 1;
    const Plan p = plan_of(n, rows, static_cast<int>(dim), used_ve);
    bool ok;
    size_t used;
    GradArgs a = carve(p, n, rows, static_cast<int>(dim), ws, ws_bytes, &ok, &used);
    if (!ok) return SPARC_ERR_WS;
    a.ids = ids;
    a.g = g;
    a.out = out;
    a.n = n;
    a.rows = rows;
    a.ldg = ldg;
    a.padding = padding_idx;
    a.tiles = p.tiles;
    a.tile = p.tile;
    a.workers = p.workers;
    a.buckets = p.buckets;
    a.shift = p.shift;
    a.dim = static_cast<int>(dim);
    a.wide_ids = ids_64 ? 1 : 0;
    a.per = p.per;
    a.scale = static_cast<float>(scale);
    if (dtype == SPARC_F32) return used_ve > 1 ? launch_grad<SPARC_F32, 4>(a, p, stream) : launch_grad<SPARC_F32, 1>(a, p, stream);
    if (dtype == SPARC_BF16) return used_ve > 1 ? launch_grad<SPARC_BF16, 8>(a, p, stream) : launch_grad<SPARC_BF16, 1>(a, p, stream);
    return used_ve > 1 ? launch_grad<SPARC_F16, 8>(a, p, stream) : launch_grad<SPARC_F16, 1>(a, p, stream);
}
