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
#include <type_traits>

#include "elem.h"

namespace {

constexpr int TILE = 2048;         // tokens per workgroup of tile_counts
constexpr int MAX_BUCKETS = 2048;  // counters per wave of tile_counts
constexpr int WAVES = 4;
constexpr int BLOCK = 64 * WAVES;
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
    int64_t n, rows, ld, ldo;
    int dim, wide_ids;
    float scale;
};

__device__ __forceinline__ int64_t token(const void* ids, const int wide, const int64_t i) {
    return wide ? static_cast<const int64_t*>(ids)[i] : static_cast<const int32_t*>(ids)[i];
}

// A group of 2^lanes_log2 lanes per row, a 16-byte vector per lane (an element of rows shorter than that), slice blockIdx.y
// of the columns; TURNS rows in flight per group, neighbouring groups on neighbouring rows.  A row's last vector ends with
// the row: it overlaps the one before it and both write the same values.
constexpr int TURNS = 4;

template <int DT, int VE>
__global__ __launch_bounds__(BLOCK) void lookup_kernel(const LookupArgs a, const int lanes_log2) {
    typedef typename Elem<DT>::type T;
    const T* table = static_cast<const T*>(a.table);
    T* out = static_cast<T*>(a.out);
    const int groups = BLOCK >> lanes_log2;
    const int unit = (static_cast<int>(blockIdx.y) << lanes_log2) + (threadIdx.x & ((1 << lanes_log2) - 1));
    if (unit * VE >= a.dim) return;
    const int col = min(unit * VE, a.dim - VE);
    const int64_t first = static_cast<int64_t>(blockIdx.x) * groups * TURNS + (threadIdx.x >> lanes_log2);
    Vec<DT, VE> v[TURNS];
    int64_t id[TURNS];
#pragma unroll
    for (int k = 0; k < TURNS; ++k) {
        const int64_t row = first + k * groups;
        id[k] = row < a.n ? token(a.ids, a.wide_ids, row) : -1;
    }
#pragma unroll
    for (int k = 0; k < TURNS; ++k)
        if (id[k] >= 0 && id[k] < a.rows) v[k].load(table + id[k] * a.ld + col);
#pragma unroll
    for (int k = 0; k < TURNS; ++k) {
        const int64_t row = first + k * groups;
        if (row >= a.n) break;
        if (id[k] >= 0 && id[k] < a.rows) {
            if (a.scale != 1.f) {   // (a copy keeps the bits)
#pragma unroll
                for (int i = 0; i < VE; ++i) v[k].set(i, v[k].get(i) * a.scale);
            }
        } else {
#pragma unroll
            for (int i = 0; i < VE; ++i) v[k].set(i, __builtin_nanf(""));
        }
        v[k].store(out + row * a.ldo + col);
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
    uint32_t* tile_start;      // [tiles][buckets + 1]: where a bucket starts inside a tile
    uint2* sorted;             // [n] {place, row inside the bucket}, by bucket inside a tile
    uint2* flat;               // [n] the same, by bucket
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

// Exclusive prefix sums over counters cnt[w * stride + k] in LDS, w < waves, k < stride (a multiple of 4, 16-byte
// aligned), key by key and inside a key wave by wave; every counter becomes its start.  All threads; tot: a word per wave of
// the workgroup.  Returns the total.
__device__ uint32_t scan_counters(uint32_t* cnt, const int stride, const int waves, uint32_t* tot) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, all_waves = blockDim.x >> 6;
    const int quads = stride >> 2, each = (quads + blockDim.x - 1) / blockDim.x;
    const int q0 = min(tid * each, quads), q1 = min(q0 + each, quads);
    uint4* c4 = reinterpret_cast<uint4*>(cnt);
    uint32_t mine = 0;
    for (int q = q0; q < q1; ++q)
        for (int w = 0; w < waves; ++w) {
            const uint4 c = c4[w * quads + q];
            mine += c.x + c.y + c.z + c.w;
        }
    uint32_t upto = mine;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const uint32_t other = __shfl_up(upto, off);
        if (lane >= off) upto += other;
    }
    if (lane == 63) tot[wave] = upto;
    __syncthreads();
    uint32_t base = upto - mine, total = 0;
    for (int w = 0; w < all_waves; ++w) {
        if (w < wave) base += tot[w];
        total += tot[w];
    }
    for (int q = q0; q < q1; ++q) {
        uint4 key = make_uint4(0, 0, 0, 0);   // places of the quad's keys in all waves
        for (int w = 0; w < waves; ++w) {
            const uint4 c = c4[w * quads + q];
            key.x += c.x; key.y += c.y; key.z += c.z; key.w += c.w;
        }
        uint4 at = make_uint4(base, base + key.x, base + key.x + key.y, base + key.x + key.y + key.z);
        base = at.w + key.w;
        for (int w = 0; w < waves; ++w) {
            const uint4 c = c4[w * quads + q];
            c4[w * quads + q] = at;
            at.x += c.x; at.y += c.y; at.z += c.z; at.w += c.w;
        }
    }
    __syncthreads();
    return total;
}

constexpr int UP_FRONT = 8;   // tokens a lane of tile_counts loads at once: a wave's share of a tile

__global__ __launch_bounds__(BLOCK) void tile_counts(const GradArgs a, const int bits, const int stride) {
    extern __shared__ __align__(16) uint32_t cnt[];   // [WAVES][stride]
    __shared__ uint32_t tot[WAVES];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t t = blockIdx.x, first = t * a.tile;
    const int64_t per_wave = a.tile / WAVES;
    const int64_t lo = min(first + wave * per_wave, a.n), hi = min(first + (wave + 1) * per_wave, a.n);
    uint32_t* mine = cnt + wave * stride;
    if (t == 0 && threadIdx.x == 0) a.long_rows[0] = 0;
    int64_t id[UP_FRONT];
    auto tokens = [&](const int64_t i0) {   // -1: none, or one without a gradient
#pragma unroll
        for (int k = 0; k < UP_FRONT; ++k) {
            const int64_t i = i0 + k * 64 + lane;
            id[k] = i < hi ? token(a.ids, a.wide_ids, i) : -1;
        }
#pragma unroll
        for (int k = 0; k < UP_FRONT; ++k)
            if (id[k] >= a.rows || id[k] == a.padding) id[k] = -1;
    };
    tokens(lo);
    for (int i = threadIdx.x; i < WAVES * stride; i += BLOCK) cnt[i] = 0;
    __syncthreads();
    for (int64_t i0 = lo; i0 < hi; i0 += 64 * UP_FRONT) {
        if (i0 > lo) tokens(i0);
#pragma unroll
        for (int k = 0; k < UP_FRONT; ++k)
            if (id[k] >= 0) atomicAdd(mine + (id[k] >> a.shift), 1u);
    }
    __syncthreads();
    const uint32_t total = scan_counters(cnt, stride, WAVES, tot);
    uint32_t* starts = a.tile_start + t * (a.buckets + 1);
    for (int b = threadIdx.x; b < a.buckets; b += BLOCK) starts[b] = cnt[b];
    if (threadIdx.x == 0) starts[a.buckets] = total;
    __syncthreads();   // (wave 0 moves its counters, which are the bucket starts, on)
    for (int64_t i0 = lo; i0 < hi; i0 += 64 * UP_FRONT) {
        if (hi - lo > 64 * UP_FRONT) tokens(i0);
#pragma unroll
        for (int k = 0; k < UP_FRONT; ++k) {
            const bool ok = id[k] >= 0;
            const uint32_t b = ok ? static_cast<uint32_t>(id[k] >> a.shift) : 0u;
            uint64_t same;
            const int r = rank_among_equals(b, bits, __ballot(ok), &same);
            if (ok) {
                const uint32_t at = mine[b];
                a.sorted[first + at + r] = make_uint2(static_cast<uint32_t>(i0 + k * 64 + lane),
                                                      static_cast<uint32_t>(id[k] - (static_cast<int64_t>(b) << a.shift)));
                if (r == 0) mine[b] = at + __popcll(same);
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // the counters as the next turn's lanes find them
        }
    }
}

// Frequent tokens make a few buckets large, so a bucket has sixteen waves; they share COUNTERS words of LDS: all for one
// wave's rows when the bucket is small (one wave then ranks it), a sixteenth each otherwise.  Rows that the counters do
// not hold at once take further passes over the bucket.
constexpr int BIG_WAVES = 16;
constexpr int COUNTERS = 8192;
constexpr int ONE_WAVE = 512;   // places that one wave ranks alone
constexpr int RANK_AHEAD = 4;   // places a lane loads at once

__global__ __launch_bounds__(64 * BIG_WAVES) void bucket_rows(const GradArgs a) {
    extern __shared__ __align__(16) uint32_t lds[];   // counters [COUNTERS], run [tiles], where [tiles]
    __shared__ uint32_t tot[BIG_WAVES];
    __shared__ uint32_t before[BIG_WAVES];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t b = blockIdx.x;
    const int64_t row0 = b << a.shift;
    const int64_t in_bucket = min(static_cast<int64_t>(1) << a.shift, a.rows - row0);
    const int tiles = static_cast<int>(a.tiles);
    uint32_t* cnt = lds;
    uint32_t* run = cnt + COUNTERS;
    uint32_t* where = run + tiles;
    // the bucket's part of every tile: running totals, and the places before the bucket (its start in `place`)
    uint32_t start = 0, total = 0;
    for (int t0 = 0; t0 < tiles; t0 += 64 * BIG_WAVES) {
        const int t = t0 + tid;
        uint32_t lo = 0, len = 0;
        if (t < tiles) {
            const uint32_t* starts = a.tile_start + static_cast<int64_t>(t) * (a.buckets + 1) + b;
            lo = starts[0];
            len = starts[1] - lo;
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
        for (int w = 0; w < BIG_WAVES; ++w) {
            if (w < wave) base += tot[w];
            total += tot[w];
            start += before[w];
        }
        if (t < tiles) run[t] = base + upto - len;
        __syncthreads();
    }
    const int waves = total <= ONE_WAVE ? 1 : BIG_WAVES;
    const int slots = static_cast<int>(min(in_bucket, static_cast<int64_t>(COUNTERS / waves)));
    int row_bits = 0, top = 1;
    while ((1 << row_bits) < slots) ++row_bits;
    while (top < tiles) top <<= 1;
    const uint32_t per_wave = waves == 1 ? total : ((total + 64 * BIG_WAVES - 1) / (64 * BIG_WAVES)) * 64;
    const uint32_t lo = min(wave * per_wave, total), hi = wave < waves ? min(lo + per_wave, total) : lo;
    uint2* flat = a.flat + start;   // the bucket's places in order, once they are found in the tiles
    uint32_t done = start;          // places of the passes before this one
    for (int64_t r0 = 0; r0 < in_bucket; r0 += slots) {
        const int count = static_cast<int>(min(in_bucket - r0, static_cast<int64_t>(slots)));
        const int stride = (count + 3) & ~3;
        for (int i = tid; i < waves * stride; i += 64 * BIG_WAVES) cnt[i] = 0;
        __syncthreads();
        uint32_t* mine = cnt + wave * stride;
        for (int turn = 0; turn < 2; ++turn) {   // count, then place
            for (uint32_t j0 = lo; j0 < hi; j0 += 64 * RANK_AHEAD) {
                uint2 e[RANK_AHEAD];
                if (turn == 0 && r0 == 0) {
                    // place j of the bucket lies in the last tile whose run begins at or before j
                    int t[RANK_AHEAD] = {};
                    for (int s = top >> 1; s > 0; s >>= 1)
#pragma unroll
                        for (int k = 0; k < RANK_AHEAD; ++k)
                            if (t[k] + s < tiles && run[t[k] + s] <= j0 + k * 64 + lane) t[k] += s;
#pragma unroll
                    for (int k = 0; k < RANK_AHEAD; ++k) {
                        const uint32_t j = j0 + k * 64 + lane;
                        e[k] = make_uint2(0u, 0xffffffffu);
                        if (j < hi) e[k] = a.sorted[t[k] * a.tile + where[t[k]] + (j - run[t[k]])];
                    }
#pragma unroll
                    for (int k = 0; k < RANK_AHEAD; ++k) {
                        const uint32_t j = j0 + k * 64 + lane;
                        if (j < hi) flat[j] = e[k];   // (read back by this very lane)
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < RANK_AHEAD; ++k) {
                        const uint32_t j = j0 + k * 64 + lane;
                        e[k] = j < hi ? flat[j] : make_uint2(0u, 0xffffffffu);
                    }
                }
#pragma unroll
                for (int k = 0; k < RANK_AHEAD; ++k) {
                    const int64_t local = static_cast<int64_t>(e[k].y) - r0;
                    const bool ok = local >= 0 && local < count;
                    const uint32_t r = ok ? static_cast<uint32_t>(local) : 0u;
                    uint64_t same;
                    const int rank = rank_among_equals(r, row_bits, __ballot(ok), &same);
                    if (ok) {
                        const uint32_t at = mine[r];
                        if (turn == 1) a.place[done + at + rank] = e[k].x;
                        if (rank == 0) mine[r] = at + __popcll(same);
                    }
                    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                }
            }
            __syncthreads();
            if (turn == 0) {
                const uint32_t all = scan_counters(cnt, stride, waves, tot);
                // wave 0's counter of the next row is where this row ends
                for (int k = tid; k < count; k += 64 * BIG_WAVES) a.row_end[row0 + r0 + k] = done + (k + 1 < count ? cnt[k + 1] : all);
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
        if (col < a.dim) {
            const float* part = a.part + 2 * first * a.dim + col;
            if (wave == 0) s = part[a.dim];              // the first worker's piece begins the row: its second slot
#pragma unroll 8
            for (int64_t p = max(lo, static_cast<int64_t>(1)); p < hi; ++p) s += part[2 * p * a.dim];
        }
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

// ---- gradient of few tokens: one launch ------------------------------------------------------------------

// Up to FEW tokens a workgroup can look through all of them itself: it owns `per` consecutive rows, writes their zeros,
// collects the places of its rows in order as keys {row, place}, sorts the keys and adds up the runs.  No workspace, one
// launch instead of four dependent ones.
constexpr int FEW = 4096, PLACE_BITS = 12;
constexpr int FEW_TURNS = FEW / BLOCK;
constexpr int FEW_BLOCKS = 1024;   // rows are dealt to at most about that many workgroups
constexpr int FEW_AHEAD = 8;       // gradient rows in flight per worker

template <int DT, int VE>
__global__ __launch_bounds__(BLOCK) void few_tokens(const GradArgs a, const int lanes_log2) {
    typedef typename Elem<DT>::type T;
    extern __shared__ __align__(16) uint32_t keys[];     // a power of two of them, at least n
    __shared__ uint32_t found[FEW_TURNS * WAVES];
    __shared__ uint32_t total_found;
    __shared__ float piece[BLOCK * VE];
    __shared__ uint32_t long_runs[FEW / LONG_ROW], n_long;
    const T* g = static_cast<const T*>(a.g);
    T* out = static_cast<T*>(a.out);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int n = static_cast<int>(a.n);
    const int64_t row0 = static_cast<int64_t>(blockIdx.x) * a.per;
    const int in_block = static_cast<int>(min(static_cast<int64_t>(a.per), a.rows - row0));
    uint32_t local[FEW_TURNS];
#pragma unroll
    for (int k = 0; k < FEW_TURNS; ++k) {
        const int i = k * BLOCK + tid;
        local[k] = 0xffffffffu;
        if (k * BLOCK < n && i < n) {
            const int64_t id = token(a.ids, a.wide_ids, i);
            if (id >= row0 && id < row0 + in_block && id != a.padding) local[k] = static_cast<uint32_t>(id - row0);
        }
    }
    // zeros behind the loads
    const int lanes = 1 << lanes_log2, workers = BLOCK >> lanes_log2, worker = tid >> lanes_log2;
    const int unit = (static_cast<int>(blockIdx.y) << lanes_log2) + (tid & (lanes - 1));
    const bool mine = unit * VE < a.dim;
    const int col = mine ? min(unit * VE, a.dim - VE) : 0;
    Vec<DT, VE> zero;
#pragma unroll
    for (int i = 0; i < VE; ++i) zero.set(i, 0.f);
    if (gridDim.y == 1) {
        T* block = out + row0 * a.dim;                   // the rows are one stretch of memory
        const int64_t len = static_cast<int64_t>(in_block) * a.dim;
        for (int64_t e = static_cast<int64_t>(tid) * VE; e < len; e += BLOCK * VE) zero.store(block + min(e, len - VE));
    } else if (mine) {
        for (int r = worker; r < in_block; r += workers) zero.store(out + (row0 + r) * a.dim + col);
    }
    // places in order: turn by turn, wave by wave, lane by lane
#pragma unroll
    for (int k = 0; k < FEW_TURNS; ++k) {
        const uint64_t hits = __ballot(local[k] != 0xffffffffu);
        if (lane == 0) found[k * WAVES + wave] = __popcll(hits);
    }
    if (tid == 0) n_long = 0;
    __syncthreads();
    static_assert(FEW_TURNS * WAVES == 64, "one wave scans the counts");
    if (wave == 0) {
        const uint32_t c = found[lane];
        uint32_t upto = c;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const uint32_t other = __shfl_up(upto, off);
            if (lane >= off) upto += other;
        }
        found[lane] = upto - c;
        if (lane == 63) total_found = upto;
    }
    __syncthreads();
    const int count = static_cast<int>(total_found);
    if (count == 0) return;                              // (the whole workgroup)
#pragma unroll
    for (int k = 0; k < FEW_TURNS; ++k) {
        const bool hit = local[k] != 0xffffffffu;
        const uint64_t hits = __ballot(hit);
        if (hit) keys[found[k * WAVES + wave] + __popcll(hits & ((1ull << lane) - 1ull))] = local[k] << PLACE_BITS | (k * BLOCK + tid);
    }
    int size = 1;
    while (size < count) size <<= 1;
    for (int i = count + tid; i < size; i += BLOCK) keys[i] = 0xffffffffu;
    __syncthreads();
    if (in_block > 1) {                                  // (one row: the places are in order)
        for (int k = 2; k <= size; k <<= 1)
            for (int j = k >> 1; j > 0; j >>= 1) {
                for (int i = tid; i < size / 2; i += BLOCK) {
                    const int x = ((i & ~(j - 1)) << 1) | (i & (j - 1)), y = x | j;
                    const uint32_t p = keys[x], q = keys[y];
                    if ((p > q) == ((x & k) == 0)) {
                        keys[x] = q;
                        keys[y] = p;
                    }
                }
                __syncthreads();
            }
    }
    __builtin_amdgcn_s_waitcnt(0x0F70);                  // vmcnt(0): the zeros have left before any wave writes sums over them
    __syncthreads();
    auto same_row = [&](const int i, const uint32_t row) { return i < count && keys[i] >> PLACE_BITS == row; };
    auto add = [&](float* acc, const int from, const int to) {   // keys [from, to)
        for (int i = from; i < to; i += FEW_AHEAD) {
            Vec<DT, VE> v[FEW_AHEAD];
#pragma unroll
            for (int k = 0; k < FEW_AHEAD; ++k)
                if (i + k < to) v[k].load(g + static_cast<int64_t>(keys[i + k] & (FEW - 1)) * a.ldg + col);
#pragma unroll
            for (int k = 0; k < FEW_AHEAD; ++k)
                if (i + k < to)
#pragma unroll
                    for (int c = 0; c < VE; ++c) acc[c] += v[k].get(c);
        }
    };
    for (int i = worker; i < count; i += workers) {
        const uint32_t row = keys[i] >> PLACE_BITS;
        if (i > 0 && keys[i - 1] >> PLACE_BITS == row) continue;   // not the first of its run
        if (same_row(i + LONG_ROW, row)) {
            if ((tid & (lanes - 1)) == 0) long_runs[atomicAdd(&n_long, 1u)] = i;
            continue;
        }
        int end = i + 1;
        while (same_row(end, row)) ++end;
        if (!mine) continue;
        float acc[VE] = {};
        add(acc, i, end);
        Vec<DT, VE> v;
#pragma unroll
        for (int c = 0; c < VE; ++c) v.set(c, acc[c] * a.scale);
        v.store(out + (row0 + row) * a.dim + col);
    }
    __syncthreads();
    for (uint32_t m = 0; m < n_long; ++m) {              // a long run: every worker takes a part, joined in order
        const int first = long_runs[m];
        const uint32_t row = keys[first] >> PLACE_BITS;
        int lo = first + LONG_ROW, hi = count;           // its end
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (keys[mid] >> PLACE_BITS == row) lo = mid;
            else hi = mid;
        }
        const int each = (hi - first + workers - 1) / workers;
        float acc[VE] = {};
        if (mine) add(acc, min(first + worker * each, hi), min(first + (worker + 1) * each, hi));
#pragma unroll
        for (int c = 0; c < VE; ++c) piece[tid * VE + c] = acc[c];
        __syncthreads();
        if (worker == 0 && mine) {
            Vec<DT, VE> v;
#pragma unroll
            for (int c = 0; c < VE; ++c) {
                double s = 0.0;
                for (int w = 0; w < workers; ++w) s += piece[(w * lanes + tid) * VE + c];
                v.set(c, static_cast<float>(s) * a.scale);
            }
            v.store(out + (row0 + row) * a.dim + col);
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

// Lanes (as a power of two, at most a wave) and slices that cover `units` vectors of a row.
int lanes_for(const int64_t units, int* slices) {
    int l = 0;
    while ((1 << l) < units && l < 6) ++l;
    *slices = static_cast<int>((units + (1 << l) - 1) >> l);
    return l;
}

Plan plan_of(const int64_t n, const int64_t rows, const int dim, const int ve) {
    Plan p;
    p.tile = TILE * ceil_div(n > 0 ? n : 1, static_cast<int64_t>(TILE) * MAX_BUCKETS);   // at most MAX_BUCKETS tiles
    p.tiles = ceil_div(n, p.tile);
    // about 256 places in a bucket, no more rows than one wave's counters hold, no more buckets than tile_counts takes
    int64_t most = ceil_div(n, 256);
    if (most < ceil_div(rows, COUNTERS)) most = ceil_div(rows, COUNTERS);
    if (most > MAX_BUCKETS) most = MAX_BUCKETS;
    p.shift = 0;
    while (ceil_div(rows, static_cast<int64_t>(1) << p.shift) > most) ++p.shift;
    p.buckets = static_cast<int>(ceil_div(rows, static_cast<int64_t>(1) << p.shift));
    p.lanes_log2 = lanes_for((dim + ve - 1) / ve, &p.slices);
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
    a.sorted = c.take<uint2>(n);
    a.flat = c.take<uint2>(n);
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
    a.n = n;
    a.rows = rows;
    a.ld = ld;
    a.ldo = ldo;
    a.dim = static_cast<int>(dim);
    a.wide_ids = ids_64 ? 1 : 0;
    a.scale = static_cast<float>(scale);
    int slices;
    const int lanes_log2 = lanes_for(vectors ? ceil_div(dim, ve) : dim, &slices);
    const int64_t blocks = ceil_div(n, static_cast<int64_t>(BLOCK >> lanes_log2) * TURNS);   // at most 2^27
    return launch_lookup([&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(slices)), dim3(BLOCK), 0, stream, a, lanes_log2);
        SPARC_CHECK_LAUNCH();
        return SPARC_OK;
    }, dtype, vectors);
}

extern "C" size_t sparc_embedding_grad_workspace_bytes(int64_t n, int64_t rows, int64_t dim, int dtype) {
    if (n < 0 || rows < 0 || dim < 0 || n > SPARC_EMBEDDING_MAX || rows > SPARC_EMBEDDING_MAX || dim > SPARC_EMBEDDING_MAX_DIM ||
        dtype < SPARC_F32 || dtype > SPARC_F16)
        return 0;
    if (n <= FEW) return 256;   // (few_tokens has none)
    const int ve = elements_of_16_bytes(dtype);
    const Plan p = plan_of(n, rows, static_cast<int>(dim), dim >= ve ? ve : 1);
    bool ok;
    size_t used;
    carve(p, n, rows, static_cast<int>(dim), nullptr, 0, &ok, &used);
    return used;
}

namespace {

template <int DT, int VE>
int launch_few(const GradArgs& a, const int lanes_log2, const int slices, sparc_stream_t stream) {
    size_t keys = 1;
    while (keys < static_cast<size_t>(a.n)) keys <<= 1;
    hipLaunchKernelGGL((few_tokens<DT, VE>), dim3(static_cast<unsigned>(ceil_div(a.rows, a.per)), static_cast<unsigned>(slices)), dim3(BLOCK),
                       keys * sizeof(uint32_t), stream, a, lanes_log2);
    SPARC_CHECK_LAUNCH();
    return SPARC_OK;
}

template <int DT, int VE>
int launch_grad(const GradArgs& a, const Plan& p, sparc_stream_t stream) {
    int bits = 0;
    while ((1 << bits) < p.buckets) ++bits;
    const int stride = (p.buckets + 3) & ~3;
    if (p.tiles > 0) {
        hipLaunchKernelGGL(tile_counts, dim3(static_cast<unsigned>(p.tiles)), dim3(BLOCK),
                           static_cast<size_t>(WAVES) * stride * sizeof(uint32_t), stream, a, bits, stride);
        SPARC_CHECK_LAUNCH();
    }
    hipLaunchKernelGGL(bucket_rows, dim3(static_cast<unsigned>(p.buckets)), dim3(64 * BIG_WAVES),
                       static_cast<size_t>(COUNTERS + 2 * p.tiles) * sizeof(uint32_t), stream, a);
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
    GradArgs a = {};
    Plan p = {};
    const bool few = n <= FEW;
    if (few) {
        if (ws_bytes < 256 || (reinterpret_cast<uintptr_t>(ws) & 255)) return SPARC_ERR_WS;   // (as for more tokens)
        p.lanes_log2 = lanes_for(ceil_div(dim, used_ve), &p.slices);
        int64_t per = ceil_div(rows, FEW_BLOCKS);
        const int64_t most = static_cast<int64_t>(1) << (32 - PLACE_BITS - 1);   // keys below the padding's
        if (per > most) per = most;
        a.per = static_cast<int>(per);
    } else {
        p = plan_of(n, rows, static_cast<int>(dim), used_ve);
        bool ok;
        size_t used;
        a = carve(p, n, rows, static_cast<int>(dim), ws, ws_bytes, &ok, &used);
        if (!ok) return SPARC_ERR_WS;
        a.per = p.per;
    }
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
    a.scale = static_cast<float>(scale);
    auto run = [&](auto type, auto width) {
        constexpr int DT = decltype(type)::value, VE = decltype(width)::value;
        return few ? launch_few<DT, VE>(a, p.lanes_log2, p.slices, stream) : launch_grad<DT, VE>(a, p, stream);
    };
    using std::integral_constant;
    const integral_constant<int, 1> one;
    if (dtype == SPARC_F32) return used_ve > 1 ? run(integral_constant<int, SPARC_F32>(), integral_constant<int, 4>()) : run(integral_constant<int, SPARC_F32>(), one);
    if (dtype == SPARC_BF16) return used_ve > 1 ? run(integral_constant<int, SPARC_BF16>(), integral_constant<int, 8>()) : run(integral_constant<int, SPARC_BF16>(), one);
    return used_ve > 1 ? run(integral_constant<int, SPARC_F16>(), integral_constant<int, 8>()) : run(integral_constant<int, SPARC_F16>(), one);
}
