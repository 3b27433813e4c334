// Lookup of scaled table rows by token, and the table's gradient by sorted tokens.
//
//     out[i, :] = round(scale * table[ids[i], :])
//     dT[v, :]  = round(scale * sum over i with ids[i] = v of g[i, :])         (rows without a token: 0)
//
// Gradient.  No atomics on values, every sum in one fixed order:
//   digit_counts, digit_scatter   a stable radix sort of the tokens, one or more digits of the row number: a workgroup per
//                  tile of tokens counts the tile's digits, then ranks its tokens (ballots inside a wave, counters in LDS
//                  between waves, the other tiles' counts before it) and scatters {row, place}.  However often one
//                  token occurs, every tile is the same work.  The sort waits on latency and leaves the memory idle, so
//                  further workgroups of its launches write the table's zeros meanwhile;
//   row_sums       adds up, over the zeros.  A worker has `per` sorted places whatever the rows hold; a row of few
//                  places belongs to the worker that meets its first, a longer one is cut and leaves one partial
//                  sum per worker, or per workgroup where it has all its places,
//   join_rows      which are added in order (float64) here.  Usually nothing to do.
// Few tokens take one launch instead (few_tokens).
#include <type_traits>

#include "elem.h"

namespace {

constexpr int SORT_WAVES = 8;
constexpr int SORT_BLOCK = 64 * SORT_WAVES;
constexpr int UP_FRONT = 4;                    // tokens a lane of a sorting workgroup holds
constexpr int CHUNK = SORT_BLOCK * UP_FRONT;   // tokens a sorting workgroup ranks at once
constexpr int MOST_TILES = 256;                // every tile reads all tiles' counts
constexpr int MOST_BITS = 11;                  // of a digit
constexpr int WAVES = 4;
constexpr int BLOCK = 64 * WAVES;
constexpr int LONG_ROW = 64;       // places of the longest row that is one worker's, at most
constexpr int STAGE = 4096;        // places of a workgroup of row_sums at most
constexpr int AHEAD = 8;           // gradient rows in flight per worker

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
// STREAM, for outputs that outgrow the Infinity Cache: they leave with nontemporal stores, and the caches keep the table's
// frequent rows.  262147 bfloat16 rows of 1024 (537 MB), frequent tokens first: 106 us = 6.0 TB/s, 157 us with plain
// stores; 134 MB: 29.5 against 31.1 us, but 71.3 against 69.5 us with a pass behind it that reads the output.  Bound by
// the stores (a fill of that size runs at 6.85 TB/s).  TURNS 2 / 8: 163 / 159 us (plain stores).
constexpr int TURNS = 4;

template <int DT, int VE, bool STREAM>
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
        v[k].template store<STREAM>(out + row * a.ldo + col);
    }
}

// ---- gradient ------------------------------------------------------------------------------------------------

// Everything the launches share.
struct GradArgs {
    const void* ids;
    const void* g;
    void* out;
    int64_t n, rows, ldg, padding;
    int64_t tile;              // tokens of a tile, a multiple of CHUNK
    int tiles;
    int dim, wide_ids;
    int per;                   // places of a worker
    int group_log2;            // workers of a workgroup of row_sums, as a power of two
    int long_row;              // places of the longest row that is one worker's
    float scale;
    uint32_t* counts;          // [tiles][1 << bits]: digits of a tile
    uint2* sorted;             // [n] {row, place}; the last pass leaves the result here
    uint2* other;              // [n] the same, between passes
    uint32_t* kept;            // one word: tokens that are rows and not padding
    uint32_t* long_rows;       // [1 + 2 * most]: count, then {row, last worker}
    uint32_t* begins;          // [workers]: 1 where a worker begins the long row that goes on in the next, 0 where it is inside
    float* part;               // [2 workers][dim]
};

// The lanes of `live` whose key equals mine.
__device__ __forceinline__ uint64_t equals(const uint32_t key, const int bits, const uint64_t live) {
    uint32_t lo = static_cast<uint32_t>(live), hi = static_cast<uint32_t>(live >> 32);
#pragma unroll
    for (int b = 0; b < MOST_BITS; ++b) {
        if (b >= bits) break;
        const uint32_t mine = 0u - ((key >> b) & 1u);            // all ones where my bit is set
        const uint64_t ones = __ballot(mine != 0u);
        lo &= ~(static_cast<uint32_t>(ones) ^ mine);             // the lanes whose bit is mine
        hi &= ~(static_cast<uint32_t>(ones >> 32) ^ mine);
    }
    return static_cast<uint64_t>(hi) << 32 | lo;
}

// Zeros that a launch writes with workgroups of its own behind those that do something else: one 16-byte store per thread,
// so that the workgroups that run at once write one stretch of memory.  627 MB in a launch: 98 us with one store per thread,
// 108 with eight, 125 with a grid of 1024 workgroups that goes round (a fill by the library: 92).  Plain stores: nontemporal
// ones change 120 to 112 us at 512 MB of zeros, nothing at 627 MB and 50 to 55 us at 200 MB, where the Infinity Cache takes part
// of them.
struct Zeros {
    uint16_t* p;
    int64_t count;         // of uint16
};
constexpr int ZERO_CHUNK = SORT_BLOCK * 8;      // uint16 of a workgroup and turn
constexpr int64_t ZERO_GROUPS = 1 << 22;        // at most (a launch has fewer than 2^32 threads): more zeros take turns

__device__ __forceinline__ void write_zeros(const Zeros& z, const int64_t first, const int64_t groups) {
    typedef uint16_t mem __attribute__((ext_vector_type(8), aligned(2)));
    const mem zero = {};
    int64_t i = first * ZERO_CHUNK + threadIdx.x * 8;
    for (; i + 8 <= z.count; i += groups * ZERO_CHUNK) *reinterpret_cast<mem*>(z.p + i) = zero;
    for (; i < z.count; i += groups * ZERO_CHUNK)
        for (int64_t k = i; k < z.count && k < i + 8; ++k) z.p[k] = 0;
}

// The next UP_FRONT {row, place} of this lane, places i0 + 64 k + lane below hi; row = ~0: none.
__device__ __forceinline__ void take(const GradArgs& a, const bool first, const uint2* in, const int64_t i0, const int64_t hi, uint2* e) {
    const int lane = threadIdx.x & 63;
    if (first) {
        int64_t id[UP_FRONT];
#pragma unroll
        for (int k = 0; k < UP_FRONT; ++k) {
            const int64_t i = i0 + k * 64 + lane;
            id[k] = i < hi ? token(a.ids, a.wide_ids, i) : -1;
        }
#pragma unroll
        for (int k = 0; k < UP_FRONT; ++k) {
            const bool ok = id[k] >= 0 && id[k] < a.rows && id[k] != a.padding;
            e[k] = make_uint2(ok ? static_cast<uint32_t>(id[k]) : ~0u, static_cast<uint32_t>(i0 + k * 64 + lane));
        }
    } else {
#pragma unroll
        for (int k = 0; k < UP_FRONT; ++k) {
            const int64_t i = i0 + k * 64 + lane;
            e[k] = i < hi ? in[i] : make_uint2(~0u, 0u);
        }
    }
}

// The sort: two or three passes of a count and a scatter.  262147 tokens over 50021 rows, two passes of 8 bits: 6.0 + 10.0 us
// each; 48979 tokens over 2449029 rows, two of 11 bits: 26 us a launch with a quarter of the 627 MB of zeros in it (4.7 and
// 9 us without).  Bound by latency: of a scatter's 9 us 3.5 are the ranking (ballots: six vector instructions a bit), 2 the
// other tiles' counts, the rest start, loads and stores.  512 threads with 4 tokens each: 5.0 + 9.4 us; 8 each: 5.7 + 11.1;
// 1024 threads with 8: 7.3 + 13.6.  Sorting by buckets of rows instead (a workgroup per bucket) took 115 to 514 us where
// frequent tokens share a bucket.
// Digits of the tokens of a tile: digit = (row >> shift) & (1 << bits) - 1.
__global__ __launch_bounds__(SORT_BLOCK) void digit_counts(const GradArgs a, const Zeros z, const uint2* in, const int shift, const int bits) {
    __shared__ uint32_t cnt[1 << MOST_BITS];
    if (static_cast<int>(blockIdx.x) >= a.tiles) return write_zeros(z, blockIdx.x - a.tiles, gridDim.x - a.tiles);
    const bool first = in == nullptr;
    const int digits = 1 << bits;
    const int64_t n = first ? a.n : *a.kept;
    const int64_t lo = blockIdx.x * a.tile, hi = min(lo + a.tile, n);
    for (int i = threadIdx.x; i < digits; i += SORT_BLOCK) cnt[i] = 0;
    __syncthreads();
    for (int64_t c = lo; c < hi; c += CHUNK) {
        uint2 e[UP_FRONT];
        take(a, first, in, c + (threadIdx.x >> 6) * (64 * UP_FRONT), hi, e);
#pragma unroll
        for (int k = 0; k < UP_FRONT; ++k)
            if (e[k].x != ~0u) atomicAdd(cnt + ((e[k].x >> shift) & (digits - 1)), 1u);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < digits; i += SORT_BLOCK) a.counts[static_cast<int64_t>(blockIdx.x) * digits + i] = cnt[i];
}

__global__ __launch_bounds__(SORT_BLOCK) void digit_scatter(const GradArgs a, const Zeros z, const uint2* in, uint2* out, const int shift, const int bits) {
    extern __shared__ __align__(16) uint32_t lds[];   // base [digits], total [digits], cnt uint16 [SORT_WAVES][digits]
    __shared__ uint32_t sums[SORT_WAVES];
    if (static_cast<int>(blockIdx.x) >= a.tiles) return write_zeros(z, blockIdx.x - a.tiles, gridDim.x - a.tiles);
    const bool first = in == nullptr;
    const int digits = 1 << bits, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    static_assert(4 * SORT_BLOCK >= 1 << MOST_BITS, "a thread has four digits");
    uint32_t *base = lds, *total = lds + digits;
    uint16_t* cnt = reinterpret_cast<uint16_t*>(total + digits);
    const int64_t n = first ? a.n : *a.kept;
    const int64_t lo = blockIdx.x * a.tile, hi = min(lo + a.tile, n);
    if (lo >= hi && blockIdx.x > 0) return;
    uint2 e[UP_FRONT];
    take(a, first, in, lo + wave * (64 * UP_FRONT), hi, e);   // (under way while the counts are added up)
    // base[d]: tokens of smaller digits in all tiles, and of digit d in the tiles before this one
    for (int d = tid; d < digits; d += SORT_BLOCK) base[d] = total[d] = 0;
    __syncthreads();
    const int columns = digits >> 2, parts = SORT_BLOCK / columns;   // four digits of every `parts`-th tile to a thread
    const int column = tid & (columns - 1);
    uint4 before = make_uint4(0, 0, 0, 0), all = before;
    const uint4* counts = reinterpret_cast<const uint4*>(a.counts) + column;
    constexpr int LOADS = 8;   // in flight
    for (int t0 = tid / columns; t0 < a.tiles; t0 += LOADS * parts) {
        uint4 c[LOADS];
#pragma unroll
        for (int k = 0; k < LOADS; ++k) {
            const int t = t0 + k * parts;
            c[k] = t < a.tiles ? counts[t * columns] : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int k = 0; k < LOADS; ++k) {
            const bool earlier = t0 + k * parts < static_cast<int>(blockIdx.x);
            all.x += c[k].x; all.y += c[k].y; all.z += c[k].z; all.w += c[k].w;
            before.x += earlier ? c[k].x : 0u; before.y += earlier ? c[k].y : 0u;
            before.z += earlier ? c[k].z : 0u; before.w += earlier ? c[k].w : 0u;
        }
    }
    const uint32_t before4[4] = {before.x, before.y, before.z, before.w}, all4[4] = {all.x, all.y, all.z, all.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        atomicAdd(base + 4 * column + k, before4[k]);
        atomicAdd(total + 4 * column + k, all4[k]);
    }
    __syncthreads();
    uint32_t mine[4] = {}, sum = 0;
    if (tid < columns)
#pragma unroll
        for (int k = 0; k < 4; ++k) sum += mine[k] = total[4 * column + k];
    uint32_t upto = sum;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const uint32_t below = __shfl_up(upto, off);
        if (lane >= off) upto += below;
    }
    if (lane == 63) sums[wave] = upto;
    __syncthreads();
    uint32_t smaller = upto - sum, kept = 0;
#pragma unroll
    for (int w = 0; w < SORT_WAVES; ++w) {
        if (w < wave) smaller += sums[w];
        kept += sums[w];
    }
    if (tid < columns)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            base[4 * column + k] += smaller;
            smaller += mine[k];
        }
    if (first && blockIdx.x == 0 && tid == 0) {
        *a.kept = kept;
        a.long_rows[0] = 0;
    }
    for (int64_t c = lo; c < hi; c += CHUNK) {
        if (c > lo) take(a, first, in, c + wave * (64 * UP_FRONT), hi, e);
        uint32_t* words = reinterpret_cast<uint32_t*>(cnt);
        for (int i = tid; i < SORT_WAVES * digits / 2; i += SORT_BLOCK) words[i] = 0;
        __syncthreads();
        uint16_t* own = cnt + wave * digits;
        uint64_t same[UP_FRONT];
        uint32_t digit[UP_FRONT], at[UP_FRONT];   // at: rank among the wave's tokens of the digit
#pragma unroll
        for (int k = 0; k < UP_FRONT; ++k) {
            const bool ok = e[k].x != ~0u;
            digit[k] = ok ? (e[k].x >> shift) & (digits - 1) : 0u;
            same[k] = equals(digit[k], bits, __ballot(ok));
        }
#pragma unroll
        for (int k = 0; k < UP_FRONT; ++k) {
            const int r = __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(same[k] >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(same[k]), 0u));
            if (e[k].x != ~0u) {
                const uint32_t c0 = own[digit[k]];
                at[k] = c0 + r;
                if (r == 0) own[digit[k]] = static_cast<uint16_t>(c0 + __popcll(same[k]));
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // the counters as the next turn's lanes find them
        }
        __syncthreads();
        for (int d = tid; d < digits; d += SORT_BLOCK) {             // counters become starts inside the chunk
            uint32_t run = 0;
#pragma unroll
            for (int w = 0; w < SORT_WAVES; ++w) {
                const uint32_t c0 = cnt[w * digits + d];
                cnt[w * digits + d] = static_cast<uint16_t>(run);
                run += c0;
            }
            total[d] = run;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < UP_FRONT; ++k)
            if (e[k].x != ~0u) out[base[digit[k]] + own[digit[k]] + at[k]] = e[k];
        __syncthreads();
        for (int d = tid; d < digits; d += SORT_BLOCK) base[d] += total[d];
    }
}

// Workers are groups of `lanes` lanes (a power of two); lane u of a group owns VE columns of the slice blockIdx.y.
// STREAM: a gradient that outgrows the Infinity Cache goes by it with nontemporal loads: 262147 rows of 512 bfloat16, three
// gradients in turn, 71 -> 58 us (the same one again and again: 91 -> 99 us for the whole call).  Now 53 us = 6.0 TB/s of
// gradient and table, bound by the loads of whole rows at random places; 8 rows in flight per worker, 4: 64 us.
// Walking rows and places together, so that a worker also writes the zeros of the rows between its own, saves the second
// write of the rows that have places (1024 columns, as many rows as places: 251 against 271 us) and lost everywhere
// else (48979 places in 2449029 rows: 153 against 125 us).
constexpr int MARGIN = LONG_ROW + 1;   // places staged on both sides of a workgroup's

template <int DT, int VE, bool STREAM>
__global__ __launch_bounds__(BLOCK) void row_sums(const GradArgs a, const int lanes_log2) {
    typedef typename Elem<DT>::type T;
    extern __shared__ __align__(16) uint32_t staged[];   // the workgroup's places from place `from` on: their rows, then they
    const T* g = static_cast<const T*>(a.g);
    T* out = static_cast<T*>(a.out);
    const int tid = threadIdx.x;
    const int lanes = 1 << lanes_log2, in_group = BLOCK >> lanes_log2, u = tid & (lanes - 1);
    uint32_t *row_of = staged, *places = staged + (in_group * a.per + 2 * MARGIN);
    const int64_t all = *a.kept;
    const int64_t e0 = min(static_cast<int64_t>(blockIdx.x) * in_group * a.per, all), e1 = min(e0 + in_group * a.per, all);
    if (e0 >= e1) return;                                // (the whole workgroup)
    const int64_t from = max(e0 - MARGIN, static_cast<int64_t>(0)), to = min(e1 + MARGIN, all);
    for (int64_t k = from + tid; k < to; k += BLOCK) {
        const uint2 s = a.sorted[k];
        row_of[k - from] = s.x;
        places[k - from] = s.y;
    }
    __syncthreads();
    const int64_t worker = static_cast<int64_t>(blockIdx.x) * in_group + (tid >> lanes_log2);
    const int64_t w0 = worker * a.per, w1 = min(w0 + a.per, all);
    const int unit = (static_cast<int>(blockIdx.y) << lanes_log2) + u, col = min(unit * VE, a.dim - VE);
    // from here on: places relative to `from`
    const int n_staged = static_cast<int>(to - from);
    // Where does the row that is cut in front of place i end?  0: no row is, -1: it is a long one, otherwise its end
    auto cut = [&](const int i) {
        if (i == 0 || i == n_staged || row_of[i - 1] != row_of[i]) return 0;   // (0 and n_staged only where all places end)
        const uint32_t r = row_of[i];
        int s_lo = max(i - a.long_row - 1, 0), s_hi = i - 1;   // its first place, as far as a long row shows
        while (s_lo < s_hi) {
            const int mid = (s_lo + s_hi) >> 1;
            if (row_of[mid] < r) s_lo = mid + 1;
            else s_hi = mid;
        }
        int f_lo = i + 1, f_hi = min(i + a.long_row + 1, n_staged);   // behind its last place
        while (f_lo < f_hi) {
            const int mid = (f_lo + f_hi) >> 1;
            if (row_of[mid] <= r) f_lo = mid + 1;
            else f_hi = mid;
        }
        return f_lo - s_lo > a.long_row ? -1 : f_lo;
    };
    int i = static_cast<int>(w0 - from), i_stop = static_cast<int>(w1 - from);
    float acc[VE] = {};
    const int b0 = static_cast<int>(e0 - from), b1 = static_cast<int>(e1 - from);
    if (e0 > 0 && e1 < all && row_of[b0 - 1] == row_of[b1] && cut(b0) < 0) {   // the workgroup is inside one long row: one piece
        const bool mine = unit * VE < a.dim;
        if (mine) {
            Vec<DT, VE> ahead[AHEAD];
#pragma unroll
            for (int k = 0; k < AHEAD; ++k)
                if (i + k < i_stop) ahead[k].template load<STREAM>(g + static_cast<int64_t>(places[i + k]) * a.ldg + col);
            for (; i < i_stop; i += AHEAD)
#pragma unroll
                for (int k = 0; k < AHEAD; ++k) {
                    if (i + k >= i_stop) break;
#pragma unroll
                    for (int j = 0; j < VE; ++j) acc[j] += ahead[k].get(j);
                    if (i + k + AHEAD < i_stop) ahead[k].template load<STREAM>(g + static_cast<int64_t>(places[i + k + AHEAD]) * a.ldg + col);
                }
        }
        if (u == 0 && blockIdx.y == 0) a.begins[worker] = 0u;
        float* joined = reinterpret_cast<float*>(places + (in_group * a.per + 2 * MARGIN));   // [WAVES][lanes][VE]
#pragma unroll
        for (int k = 0; k < VE; ++k) {
            double s = acc[k];
            for (int off = lanes; off < 64; off <<= 1) s += __shfl_xor(s, off);
            if ((tid & 63) < lanes) joined[((tid >> 6) * lanes + u) * VE + k] = static_cast<float>(s);
        }
        __syncthreads();
        if (tid < lanes && mine) {
            float* p = a.part + 2 * worker * a.dim + col;
#pragma unroll
            for (int k = 0; k < VE; ++k) {
                double s = 0.0;
                for (int w = 0; w < WAVES; ++w) s += joined[(w * lanes + u) * VE + k];
                p[k] = static_cast<float>(s);
            }
        }
        return;
    }
    if (w0 >= w1 || unit * VE >= a.dim) return;          // no barrier below
    int c = cut(i);
    bool inside = c < 0;                                 // a long row that began in an earlier worker
    if (c > 0) i = c;                                    // an earlier worker has the whole row
    c = cut(i_stop);
    const bool goes_on = c < 0;                          // a long row goes on in the next worker
    if (c > 0) i_stop = c;                               // the row that is cut here is this worker's
    if (i >= i_stop) return;
    uint32_t row = row_of[i];
    auto finish_row = [&]() {
        if (inside) {
            float* p = a.part + (2 * worker) * a.dim + col;
#pragma unroll
            for (int k = 0; k < VE; ++k) p[k] = acc[k];
            if (u == 0 && blockIdx.y == 0) {             // the last piece of a long row: announce it
                const uint32_t at = atomicAdd(a.long_rows, 1u);
                a.long_rows[1 + 2 * at] = row;
                a.long_rows[2 + 2 * at] = static_cast<uint32_t>(worker);
            }
            inside = false;
        } else {
            Vec<DT, VE> v;
#pragma unroll
            for (int k = 0; k < VE; ++k) v.set(k, acc[k] * a.scale);
            v.store(out + static_cast<int64_t>(row) * a.dim + col);
        }
#pragma unroll
        for (int k = 0; k < VE; ++k) acc[k] = 0.f;
    };
    Vec<DT, VE> ahead[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
        if (i + k < i_stop) ahead[k].template load<STREAM>(g + static_cast<int64_t>(places[i + k]) * a.ldg + col);
    while (i < i_stop) {
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            if (i + k >= i_stop) break;
            if (row_of[i + k] != row) {
                finish_row();
                row = row_of[i + k];
            }
#pragma unroll
            for (int j = 0; j < VE; ++j) acc[j] += ahead[k].get(j);
            if (i + k + AHEAD < i_stop) ahead[k].template load<STREAM>(g + static_cast<int64_t>(places[i + k + AHEAD]) * a.ldg + col);
        }
        i += AHEAD;
    }
    if (!goes_on) {
        finish_row();
    } else {
        if (u == 0 && blockIdx.y == 0) a.begins[worker] = inside ? 0u : 1u;
        float* p = a.part + (2 * worker + (inside ? 0 : 1)) * a.dim + col;
#pragma unroll
        for (int k = 0; k < VE; ++k) p[k] = acc[k];
    }
}

// Long rows: slice blockIdx.y of 64 columns, VE (four, or one where a row has fewer) columns to a lane.  The pieces of a
// row are dealt to the groups of 16 lanes, which have JOIN_AHEAD of them in flight; the groups' sums meet in their order.
// Where there are far fewer rows than workgroups, four of these share a slice, in groups of 4 lanes: 262147 places of 512
// bfloat16 all the same 131 -> 98 us (always: frequent tokens first 102 -> 121).
// 9 us for the 300 long rows of 262147 tokens, frequent ones first; 4.6 us (the wait for the launch before) for none.
constexpr int JOIN_THREADS = 256, JOIN_COLS = 64, JOIN_AHEAD = 8;

template <int DT, int VE>
__global__ __launch_bounds__(JOIN_THREADS) void join_rows(const GradArgs a) {
    typedef typename Elem<DT>::type T;
    __shared__ double sum[JOIN_THREADS * VE];            // [groups][cols]
    __shared__ int begun;
    const uint32_t count = a.long_rows[0];
    const int parts_log2 = VE > 1 && 4 * count <= gridDim.x ? 2 : 0;
    const int lanes_log2 = 4 - parts_log2, groups = JOIN_THREADS >> lanes_log2, cols = VE << lanes_log2;
    static_assert(JOIN_COLS == 4 << 4, "a slice is 16 lanes of four columns");
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, group = threadIdx.x >> lanes_log2;
    for (uint32_t k = blockIdx.x; k < count << parts_log2; k += gridDim.x) {
        const int base = blockIdx.y * JOIN_COLS + (k & ((1u << parts_log2) - 1u)) * cols;
        const int unit = base + (threadIdx.x & ((1 << lanes_log2) - 1)) * VE, col = max(min(unit, a.dim - VE), 0);
        const int64_t row = a.long_rows[1 + 2 * (k >> parts_log2)];
        const int last = a.long_rows[2 + 2 * (k >> parts_log2)];
        if (wave == 0) {                                 // the worker that began the row: near by, or found by the row's first place
            const int before = last - 1 - lane;
            const uint64_t found = __ballot(before >= 0 && a.begins[max(before, 0)] == 1u);
            int worker = last - __ffsll(static_cast<unsigned long long>(found));
            if (found == 0) {
                int64_t lo = 0, hi = *a.kept;
                while (hi > lo) {
                    const int64_t width = (hi - lo + 63) >> 6, e = lo + lane * width;
                    const int smaller = __popcll(__ballot(e < hi && a.sorted[e].x < row));
                    if (smaller == 0) break;
                    hi = min(hi, lo + smaller * width);
                    lo += (smaller - 1) * width + 1;
                }
                worker = static_cast<int>(lo / a.per);
            }
            if (lane == 0) begun = worker;
        }
        __syncthreads();
        const int first = begun;
        // a piece per worker, but one for all workers of a workgroup that is wholly inside the row; the first worker's piece
        // begins the row: its second slot
        const int g0 = first >> a.group_log2, g1 = last >> a.group_log2;
        const int head = g0 == g1 ? last - first + 1 : ((g0 + 1) << a.group_log2) - first, inner = g0 == g1 ? head : head + g1 - g0 - 1;
        const int pieces = g0 == g1 ? head : inner + last - (g1 << a.group_log2) + 1;
        auto piece = [&](const int p) {
            const int worker = p < head ? first + p : p < inner ? (g0 + 1 + p - head) << a.group_log2 : (g1 << a.group_log2) + (p - inner);
            return a.part + (2 * static_cast<int64_t>(worker) + (p == 0 ? 1 : 0)) * a.dim + col;
        };
        double s[VE] = {};
        if (unit < a.dim) {
            for (int p0 = group; p0 < pieces; p0 += groups * JOIN_AHEAD) {
                Vec<SPARC_F32, VE> v[JOIN_AHEAD];
#pragma unroll
                for (int j = 0; j < JOIN_AHEAD; ++j) {
                    const int p = p0 + j * groups;
                    if (p < pieces) v[j].load(piece(p));
                }
#pragma unroll
                for (int j = 0; j < JOIN_AHEAD; ++j)
                    if (p0 + j * groups < pieces)
#pragma unroll
                        for (int c = 0; c < VE; ++c) s[c] += v[j].get(c);
            }
#pragma unroll
            for (int c = 0; c < VE; ++c)
                if (col + c >= base) sum[group * cols + col + c - base] = s[c];
        }
        __syncthreads();
        const int mine = base + threadIdx.x;
        if (threadIdx.x < cols && mine < a.dim) {
            double all = 0.0;
#pragma unroll 16
            for (int w = 0; w < groups; ++w) all += sum[w * cols + threadIdx.x];
            static_cast<T*>(a.out)[row * a.dim + mine] = Elem<DT>::down(static_cast<float>(all) * a.scale);
        }
        __syncthreads();
    }
}

// ---- gradient of few tokens: one launch ------------------------------------------------------------------

// Up to FEW tokens a workgroup can look through all of them itself: it writes the zeros of its rows, collects their places
// as keys {row, place}, sorts the keys by row and adds up the runs.  No workspace, one launch instead of six dependent
// ones.  The rows are dealt out in turn, in groups of at least GROUP_BYTES, because frequent tokens are often neighbours.
// A workgroup may get all tokens as well as none: the keys are collected in an order fixed by the tokens, so that a radix
// sort of the row alone will do, and dealt to the workers in equal shares, of which one long run has many.
//
// Measured, a call in us for uniform tokens, frequent first, all the same: 2437 tokens over 2708 rows of 64 floats 8.9, 11.2,
// 21 (the sort takes 26 for the first); 8192 over 50000 rows of 64 floats 11.7, 16.3, 57 (9000 tokens by the sort: 30, 40, 38);
// 8192 of 512 floats 27, 33, 76 (by the sort 40, 49, 55), of 2048 floats 100, 108, 201 (105, 110, 113): beyond 16 MiB of
// gradient the sort.  Bound by the chain tokens -> keys -> rows -> stores, and where all tokens are the same by what one CU
// reads, 45 GB/s; hence workers of at most 16 lanes, so that wider rows have several workgroups: 4096 of 512 bfloat16 all the
// same 111 -> 44 us, uniform 14.4 -> 15.2; 8 lanes 33 and 16.2.  FEW_LONG 16, 32: frequent first 17.3, 17.7; FEW_AHEAD 4, 16:
// all the same 66, 54, uniform 11.7, 12.6.  With a bitonic sort of all keys and long runs one by one: 8192 tokens over 300
// rows of one float, frequent first, 306 us, now 20.
constexpr int FEW = 8192, PLACE_BITS = 13;
constexpr int64_t FEW_BYTES = 16 << 20;   // of gradient
constexpr int64_t FEW_ROW_BYTES = 32768;
constexpr int FEW_WAVES = 8, FEW_THREADS = 64 * FEW_WAVES;
constexpr int FEW_TOKENS = FEW / FEW_THREADS;   // of a thread
constexpr int FEW_BLOCKS_LOG2 = 9;   // workgroups that the rows are dealt to, all slices together
constexpr int FEW_AHEAD = 8;         // gradient rows in flight per worker
constexpr int FEW_LONG = 8;         // places of the longest run that is one worker's
constexpr int FEW_BITS = 8;          // of a digit of the radix sort
constexpr int FEW_LANES_LOG2 = 4;    // of a worker at most: slices of 256 bytes
constexpr int GROUP_BYTES = 16 << FEW_LANES_LOG2;   // (rows narrower than that are one slice)

// Row r belongs to workgroup (r >> group) mod 2^blocks, where it is row local(r).
struct Dealt {
    int group, blocks, bits;   // bits: of a local row
    __device__ __forceinline__ uint32_t block_of(const uint32_t r) const { return (r >> group) & ((1u << blocks) - 1u); }
    __device__ __forceinline__ uint32_t local(const uint32_t r) const {
        return (r >> group >> blocks) << group | (r & ((1u << group) - 1u));
    }
    __device__ __forceinline__ int64_t row(const uint32_t block, const uint32_t local) const {
        return ((static_cast<int64_t>(local >> group) << blocks | block) << group) | (local & ((1u << group) - 1u));
    }
};

// The keys of this workgroup's tokens, in the order of (wave, turn, element, lane), whatever the type; returns how many.
template <typename ID>
__device__ __forceinline__ int collect_rows(const ID* ids, const int n, const int64_t rows, const int64_t padding, const Dealt dealt,
                                            uint32_t* keys, uint32_t* found) {
    constexpr int VE = 4, TURNS = FEW_TOKENS / VE;
    typedef ID mem __attribute__((ext_vector_type(VE), aligned(sizeof(ID))));
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    auto place = [](const int k, const int c) { return (k * FEW_THREADS + static_cast<int>(threadIdx.x)) * VE + c; };
    mem v[TURNS];
#pragma unroll
    for (int k = 0; k < TURNS; ++k) {
        if (k * FEW_THREADS * VE >= n) break;
        const int i = place(k, 0);
        if (i + VE <= n) {
            v[k] = *reinterpret_cast<const mem*>(ids + i);
        } else {
#pragma unroll
            for (int c = 0; c < VE; ++c) v[k][c] = i + c < n ? ids[i + c] : static_cast<ID>(-1);
        }
    }
    uint32_t hits = 0;
    int count = 0;
#pragma unroll
    for (int k = 0; k < TURNS; ++k) {
        if (k * FEW_THREADS * VE >= n) break;
#pragma unroll
        for (int c = 0; c < VE; ++c) {
            const int64_t id = v[k][c];
            const bool hit = dealt.block_of(static_cast<uint32_t>(id)) == blockIdx.x && id >= 0 && id < rows && id != padding;
            hits |= hit ? 1u << (k * VE + c) : 0u;
            count += __popcll(__ballot(hit));
        }
    }
    if (lane == 0) found[wave] = count;
    __syncthreads();
    int at = 0, total = 0;
#pragma unroll
    for (int w = 0; w < FEW_WAVES; ++w) {
        if (w < wave) at += found[w];
        total += found[w];
    }
    total = __builtin_amdgcn_readfirstlane(total);
    if (count > 0)
#pragma unroll
        for (int k = 0; k < TURNS; ++k) {
            if (k * FEW_THREADS * VE >= n) break;
#pragma unroll
            for (int c = 0; c < VE; ++c) {
                const bool hit = hits >> (k * VE + c) & 1u;
                const uint64_t here = __ballot(hit);
                if (here == 0) continue;
                if (hit)
                    keys[at + __popcll(here & ((1ull << lane) - 1ull))] =
                        dealt.local(static_cast<uint32_t>(v[k][c])) << PLACE_BITS | static_cast<uint32_t>(place(k, c));
                at += __popcll(here);
            }
        }
    return total;
}

// By row and place, up to a key per thread: every key counts the smaller ones.  (Bitonic: 10 to 45 barriers.)
__device__ __forceinline__ void rank_sort(uint32_t* keys, const int count) {
    const int tid = threadIdx.x;
    if (count <= 64) {
        if (tid >= 64) return;
        const uint32_t key = tid < count ? keys[tid] : ~0u;
        int rank = 0;
        for (int j = 0; j < count; ++j) rank += __builtin_amdgcn_readlane(static_cast<int>(key), j) < static_cast<int>(key) ? 1 : 0;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // read by all before any writes
        if (tid < count) keys[rank] = key;
        return;
    }
    const int fours = (count + 3) >> 2;
    if (tid < 4 * fours - count) keys[count + tid] = ~0u;
    __syncthreads();
    const uint32_t key = tid < count ? keys[tid] : 0u;
    uint32_t rank = 0;
    if ((tid & ~63) < count)
#pragma unroll 4
        for (int j = 0; j < fours; ++j) {
            const uint4 k = reinterpret_cast<const uint4*>(keys)[j];
            rank += (k.x < key ? 1u : 0u) + (k.y < key ? 1u : 0u) + (k.z < key ? 1u : 0u) + (k.w < key ? 1u : 0u);
        }
    __syncthreads();
    if (tid < count) keys[rank] = key;
}

// By row, keys of a row as they came.  cnt: [FEW_WAVES][1 << FEW_BITS], sums: [FEW_WAVES].
__device__ __forceinline__ void radix_sort(uint32_t* keys, const int count, const int row_bits, uint16_t* cnt, uint32_t* sums) {
    constexpr int DIGITS = 1 << FEW_BITS;
    static_assert(DIGITS <= FEW_THREADS && FEW_BITS <= MOST_BITS, "a digit per thread");
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int steps = (count + FEW_THREADS - 1) / FEW_THREADS;   // keys of a lane
    const int from = wave * steps * 64 + lane;
    uint16_t* own = cnt + wave * DIGITS;
    for (int shift = PLACE_BITS; shift < PLACE_BITS + row_bits; shift += FEW_BITS) {
        uint32_t e[FEW_TOKENS], at[FEW_TOKENS];   // at: rank among the wave's keys of the digit
#pragma unroll
        for (int k = 0; k < FEW_TOKENS; ++k)
            if (k < steps) e[k] = from + k * 64 < count ? keys[from + k * 64] : 0u;
        for (int i = tid; i < FEW_WAVES * DIGITS / 2; i += FEW_THREADS) reinterpret_cast<uint32_t*>(cnt)[i] = 0;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < FEW_TOKENS; ++k) {
            if (k >= steps) break;
            const bool ok = from + k * 64 < count;
            const uint32_t digit = (e[k] >> shift) & (DIGITS - 1);
            const uint64_t same = equals(digit, FEW_BITS, __ballot(ok));
            const int r = __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(same >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(same), 0u));
            if (ok) {
                const uint32_t c0 = own[digit];
                at[k] = c0 + r;
                if (r == 0) own[digit] = static_cast<uint16_t>(c0 + __popcll(same));
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // the counters as the next turn's lanes find them
        }
        __syncthreads();
        uint32_t of_digit = 0, upto = 0;
        if (tid < DIGITS) {
#pragma unroll
            for (int w = 0; w < FEW_WAVES; ++w) of_digit += cnt[w * DIGITS + tid];
            upto = of_digit;
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) {
                const uint32_t below = __shfl_up(upto, off);
                if (lane >= off) upto += below;
            }
            if (lane == 63) sums[wave] = upto;
        }
        __syncthreads();
        if (tid < DIGITS) {
            uint32_t run = upto - of_digit;
#pragma unroll
            for (int w = 0; w < DIGITS / 64; ++w)
                if (w < wave) run += sums[w];
#pragma unroll
            for (int w = 0; w < FEW_WAVES; ++w) {
                const uint32_t c0 = cnt[w * DIGITS + tid];
                cnt[w * DIGITS + tid] = static_cast<uint16_t>(run);
                run += c0;
            }
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < FEW_TOKENS; ++k)
            if (k < steps && from + k * 64 < count) keys[own[(e[k] >> shift) & (DIGITS - 1)] + at[k]] = e[k];
        __syncthreads();
    }
}

__global__ __launch_bounds__(SORT_BLOCK) void zeros_kernel(const Zeros z) { write_zeros(z, blockIdx.x, gridDim.x); }

// zeros: write them here, too.  64 to 66 registers, or a third workgroup would wait for a whole round: 4101 tokens over 451 rows of 359
// floats, 768 workgroups, 21.7 us with 84 registers, 15.6 with 64, 14.4 with 384 workgroups.
template <int DT, int VE>
__global__ __launch_bounds__(FEW_THREADS, 6) void few_tokens(const GradArgs a, const Dealt dealt, const int lanes_log2, const bool zeros) {
    typedef typename Elem<DT>::type T;
    extern __shared__ __align__(16) uint32_t keys[];     // n, and up to a multiple of four
    __shared__ uint32_t sums[FEW_WAVES];
    // counters of the sort, then sums of the workers' pieces
    __shared__ __align__(16) uint32_t shared[VE > 2 ? FEW_THREADS * VE : FEW_THREADS * 2];
    static_assert(sizeof(shared) >= sizeof(uint16_t) * FEW_WAVES << FEW_BITS, "the sort's counters fit");
    float* piece = reinterpret_cast<float*>(shared);
    const T* g = static_cast<const T*>(a.g);
    T* out = static_cast<T*>(a.out);
    const int tid = threadIdx.x;
    const int n = static_cast<int>(a.n);
    const int lanes = 1 << lanes_log2, workers = FEW_THREADS >> lanes_log2, worker = tid >> lanes_log2;
    const int unit = (static_cast<int>(blockIdx.y) << lanes_log2) + (tid & (lanes - 1));
    const bool mine = unit * VE < a.dim;
    const int col = mine ? min(unit * VE, a.dim - VE) : 0;
    Vec<DT, VE> zero;
#pragma unroll
    for (int i = 0; i < VE; ++i) zero.set(i, 0.f);
    if (!zeros) {
    } else if (dealt.group > 0) {                        // narrow rows, one slice: a group of them is one stretch of memory
        const int64_t stretch = static_cast<int64_t>(a.dim) << dealt.group, len = a.rows * a.dim;
        const int per_stretch = static_cast<int>((stretch + VE - 1) / VE);
        int log2 = 0;
        while ((1 << log2) < per_stretch) ++log2;        // (at most FEW_THREADS: a stretch is shorter than 2 GROUP_BYTES)
        const int e = (tid & ((1 << log2) - 1)) * VE;
        for (int64_t q = tid >> log2;; q += FEW_THREADS >> log2) {
            const int64_t from = ((q << dealt.blocks) + blockIdx.x) * stretch;
            if (from >= len) break;
            const int64_t here = min(stretch, len - from);
            if (e < here) zero.store(out + from + min(static_cast<int64_t>(e), here - VE));
        }
    } else if (mine) {
        for (int64_t r = blockIdx.x + (static_cast<int64_t>(worker) << dealt.blocks); r < a.rows; r += static_cast<int64_t>(workers) << dealt.blocks)
            zero.store(out + r * a.dim + col);
    }
    const int count = a.wide_ids ? collect_rows(static_cast<const int64_t*>(a.ids), n, a.rows, a.padding, dealt, keys, sums)
                                 : collect_rows(static_cast<const int32_t*>(a.ids), n, a.rows, a.padding, dealt, keys, sums);
    if (count == 0) return;                              // (the whole workgroup)
    __syncthreads();
    if (count <= FEW_THREADS) {
        rank_sort(keys, count);
    } else {
        bool in_order = true;
        for (int i = tid + 1; i < count; i += FEW_THREADS) in_order &= keys[i - 1] >> PLACE_BITS <= keys[i] >> PLACE_BITS;
        if (!__syncthreads_and(in_order)) radix_sort(keys, count, dealt.bits, reinterpret_cast<uint16_t*>(shared), sums);
    }
    __builtin_amdgcn_s_waitcnt(0x0F70);                  // vmcnt(0): the zeros have left before any wave writes sums over them
    __syncthreads();
    auto row_at = [&](const int i) { return keys[i] >> PLACE_BITS; };
    // behind the last key of the run that key i is in (the keys up to `last` are looked at)
    auto end_of = [&](const int i, int last) {
        const uint32_t row = row_at(i);
        int end = i + 1;
        while (end < last) {
            const int mid = (end + last) >> 1;
            if (row_at(mid) == row) end = mid + 1;
            else last = mid;
        }
        return end;
    };
    // The workers' shares.  A run of at most FEW_LONG keys belongs to the worker that meets its first; a longer one is cut.
    // Where does the run that is cut in front of key i end?  0: none is, -1: it is a long one.
    auto cut = [&](const int i) {
        if (i == 0 || i >= count || row_at(i - 1) != row_at(i)) return 0;
        const uint32_t row = row_at(i);
        int begin = max(i - FEW_LONG - 1, 0), here = i - 1;
        while (begin < here) {
            const int mid = (begin + here) >> 1;
            if (row_at(mid) != row) begin = mid + 1;
            else here = mid;
        }
        const int end = end_of(i, min(i + FEW_LONG + 1, count));
        return end - begin > FEW_LONG ? -1 : end;
    };
    const int per = (count + workers - 1) / workers;
    int i = min(worker * per, count), stop = min(i + per, count);
    int c = i < stop ? cut(i) : 0;
    bool inside = c < 0;                                 // a long run that began in an earlier worker
    if (c > 0) i = c;
    c = i < stop ? cut(stop) : 0;
    const bool goes_on = c < 0;                          // a long run goes on in the next worker
    if (c > 0) stop = c;
    float acc[VE] = {};
    bool begun = false;                                  // and it began here: this worker adds up its pieces
    uint32_t row = 0;
    auto store = [&](const uint32_t local) {
        Vec<DT, VE> v;
#pragma unroll
        for (int k = 0; k < VE; ++k) v.set(k, acc[k] * a.scale);
        v.store(out + dealt.row(blockIdx.x, local) * a.dim + col);
    };
    auto leave = [&]() {                                 // a piece of a long run
#pragma unroll
        for (int k = 0; k < VE; ++k) piece[tid * VE + k] = acc[k];
    };
    if (mine && i < stop) {
        row = row_at(i);
        auto load = [&](Vec<DT, VE>& v, const int k) {
            v.load(g + static_cast<int64_t>(keys[k] & ((1 << PLACE_BITS) - 1)) * a.ldg + col);
        };
        Vec<DT, VE> ahead[FEW_AHEAD];
#pragma unroll
        for (int k = 0; k < FEW_AHEAD; ++k)
            if (i + k < stop) load(ahead[k], i + k);
        for (; i < stop; i += FEW_AHEAD) {
#pragma unroll
            for (int k = 0; k < FEW_AHEAD; ++k) {
                if (i + k >= stop) break;
                if (row_at(i + k) != row) {
                    if (inside) leave();
                    else store(row);
                    inside = false;
                    row = row_at(i + k);
#pragma unroll
                    for (int j = 0; j < VE; ++j) acc[j] = 0.f;
                }
#pragma unroll
                for (int j = 0; j < VE; ++j) acc[j] += ahead[k].get(j);
                if (i + k + FEW_AHEAD < stop) load(ahead[k], i + k + FEW_AHEAD);
            }
        }
        if (inside) leave();
        else if (goes_on) begun = true;
        else store(row);
    }
    __syncthreads();
    if (begun) {
        const int last = (end_of(stop - 1, count) - 1) / per;
        double s[VE];
#pragma unroll
        for (int k = 0; k < VE; ++k) s[k] = acc[k];
#pragma unroll 8
        for (int w = worker + 1; w <= last; ++w)
#pragma unroll
            for (int k = 0; k < VE; ++k) s[k] += piece[(tid + ((w - worker) << lanes_log2)) * VE + k];
#pragma unroll
        for (int k = 0; k < VE; ++k) acc[k] = static_cast<float>(s[k]);
        store(row);
    }
}

// Sizes of the launches and of the workspace's parts, from n, rows and dim alone.
struct Plan {
    int64_t tile, workers;
    int tiles, passes, bits, per, long_row, lanes_log2, slices, in_group;
};

int64_t ceil_div(const int64_t a, const int64_t b) { return (a + b - 1) / b; }

// Lanes (as a power of two, at most a wave) and slices that cover `units` vectors of a row.
int lanes_for(const int64_t units, int* slices, const int most_log2 = 6) {
    int l = 0;
    while ((1 << l) < units && l < most_log2) ++l;
    *slices = static_cast<int>((units + (1 << l) - 1) >> l);
    return l;
}

Plan plan_of(const int64_t n, const int64_t rows, const int dim, const int ve) {
    Plan p;
    p.tile = CHUNK * ceil_div(n, static_cast<int64_t>(CHUNK) * MOST_TILES);
    p.tiles = static_cast<int>(ceil_div(n, p.tile));
    int bits = 2;
    while ((static_cast<int64_t>(1) << bits) < rows) ++bits;
    // wide digits save passes, but every tile reads the counts of all digits of all tiles
    const int most = p.tiles <= 32 ? MOST_BITS : 8;
    p.passes = (bits + most - 1) / most;
    p.bits = (bits + p.passes - 1) / p.passes;
    p.lanes_log2 = lanes_for((dim + ve - 1) / ve, &p.slices);
    p.in_group = BLOCK >> p.lanes_log2;
    // places of a worker: enough workers for every SIMD's wave slots first, up to 64 places then
    const int64_t wanted = ceil_div(n, static_cast<int64_t>(8192) * 64 >> p.lanes_log2);
    p.per = static_cast<int>(wanted < 8 ? 8 : wanted > 64 ? 64 : wanted);
    if (static_cast<int64_t>(p.per) * p.in_group > STAGE) p.per = STAGE / p.in_group;
    p.workers = ceil_div(n, p.per);
    // Two shares, or a worker that has a whole row would be the last by far (per is 8 to 64).  Always 64, always 16: 20000 places over 5000 rows of 64 floats, frequent first, 41, 34 us; 1000000 over 50000, uniform, 99, 488.
    p.long_row = 2 * p.per > LONG_ROW ? LONG_ROW : 2 * p.per;
    return p;
}

template <int DT, int VE>
int launch_lookup(LookupArgs a, sparc_stream_t stream) {
    typedef typename Elem<DT>::type T;
    int slices;
    const int lanes_log2 = lanes_for(ceil_div(a.dim, VE), &slices);
    const bool streaming = a.n * a.dim * static_cast<int64_t>(sizeof(T)) > SPARC_KEEP_BYTES;
    const int64_t rows_of_block = static_cast<int64_t>(BLOCK >> lanes_log2) * TURNS;
    const int64_t most = static_cast<int64_t>(UINT32_MAX / BLOCK) * rows_of_block;   // a launch has fewer than 2^32 threads along x
    for (int64_t left = a.n; left > 0; left -= most) {
        a.n = left < most ? left : most;
        const dim3 grid(static_cast<unsigned>(ceil_div(a.n, rows_of_block)), static_cast<unsigned>(slices));
        if (streaming) hipLaunchKernelGGL((lookup_kernel<DT, VE, true>), grid, dim3(BLOCK), 0, stream, a, lanes_log2);
        else hipLaunchKernelGGL((lookup_kernel<DT, VE, false>), grid, dim3(BLOCK), 0, stream, a, lanes_log2);
        SPARC_CHECK_LAUNCH();
        a.ids = static_cast<const char*>(a.ids) + a.n * (a.wide_ids ? 8 : 4);
        a.out = static_cast<T*>(a.out) + a.n * a.ldo;
    }
    return SPARC_OK;
}

// f(type, width): the element type and the elements of a vector as integral constants.
template <typename F>
int dispatch(const int dtype, const int64_t dim, F&& f) {
    using std::integral_constant;
    const integral_constant<int, 1> one;
    if (dtype == SPARC_F32) return dim >= 4 ? f(integral_constant<int, SPARC_F32>(), integral_constant<int, 4>()) : f(integral_constant<int, SPARC_F32>(), one);
    if (dtype == SPARC_BF16) return dim >= 8 ? f(integral_constant<int, SPARC_BF16>(), integral_constant<int, 8>()) : f(integral_constant<int, SPARC_BF16>(), one);
    return dim >= 8 ? f(integral_constant<int, SPARC_F16>(), integral_constant<int, 8>()) : f(integral_constant<int, SPARC_F16>(), one);
}

GradArgs carve(const Plan& p, const int64_t n, const int dim, void* ws, const size_t ws_bytes, bool* ok, size_t* used) {
    GradArgs a = {};
    WsCarver c(ws, ws_bytes);
    a.counts = c.take<uint32_t>(static_cast<size_t>(p.tiles) << p.bits);
    a.sorted = c.take<uint2>(n);
    a.other = c.take<uint2>(p.passes > 1 ? n : 0);
    a.kept = c.take<uint32_t>(1);
    a.long_rows = c.take<uint32_t>(1 + 2 * (n / p.long_row + 1));
    a.begins = c.take<uint32_t>(p.workers);
    a.part = c.take<float>(static_cast<size_t>(2) * p.workers * dim);
    *ok = c.ok();
    *used = c.off;
    return a;
}

// Rows in very many slices make many workgroups that all look through the tokens.  30 tokens over 300 rows, uniform and all the
// same, in one launch and by the sort: of 4096 floats 9.1, 15.8 and 18.3, 20.4 us; of 8192 14.5, 28 and 18.8, 24.5; of 16384
// 23, 50 and 19.5, 32.
bool few_enough(const int64_t n, const int64_t dim, const int dtype) {
    const int64_t row_bytes = dim * (dtype == SPARC_F32 ? 4 : 2);
    return n <= FEW && row_bytes <= FEW_ROW_BYTES && n * row_bytes <= FEW_BYTES;
}

int elements_of_16_bytes(const int dtype) { return dtype == SPARC_F32 ? 4 : 8; }

}  // namespace

extern "C" int sparc_embedding_fwd(int64_t n, int64_t rows, int64_t dim, int dtype, const void* ids, int ids_64, const void* table,
                                   int64_t ld, double scale, void* out, int64_t ldo, sparc_stream_t stream) {
    if (n < 0 || rows < 0 || dim < 0 || dtype < SPARC_F32 || dtype > SPARC_F16 || ld < dim || ldo < dim || !ids || !out || (rows > 0 && !table))
        return SPARC_ERR_ARG;
    if (n > SPARC_EMBEDDING_MAX || rows > SPARC_EMBEDDING_MAX || dim > SPARC_EMBEDDING_MAX_DIM) return SPARC_ERR_SIZE;
    if (n == 0 || dim == 0) return SPARC_OK;
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
    return dispatch(dtype, dim, [&](auto type, auto width) { return launch_lookup<decltype(type)::value, decltype(width)::value>(a, stream); });
}

extern "C" size_t sparc_embedding_grad_workspace_bytes(int64_t n, int64_t rows, int64_t dim, int dtype) {
    if (n < 0 || rows < 0 || dim < 0 || n > SPARC_EMBEDDING_MAX || rows > SPARC_EMBEDDING_MAX || dim > SPARC_EMBEDDING_MAX_DIM ||
        dtype < SPARC_F32 || dtype > SPARC_F16)
        return 0;
    if (n == 0 || few_enough(n, dim, dtype)) return 0;
    const int ve = elements_of_16_bytes(dtype);
    const Plan p = plan_of(n, rows, static_cast<int>(dim), dim >= ve ? ve : 1);
    bool ok;
    size_t used;
    carve(p, n, static_cast<int>(dim), nullptr, 0, &ok, &used);
    return used;
}

namespace {

template <int DT, int VE>
int launch_grad(const GradArgs& a, const Plan& p, sparc_stream_t stream) {
    const int64_t half_words = a.rows * a.dim * static_cast<int64_t>(sizeof(typename Elem<DT>::type)) / 2;
    const size_t lds = (static_cast<size_t>(1) << p.bits) * (2 * sizeof(uint32_t) + SORT_WAVES * sizeof(uint16_t));
    // the zeros are dealt to the launches of the sort
    const int64_t chunks = ceil_div(half_words, ZERO_CHUNK), each = ceil_div(chunks, 2 * p.passes);
    int64_t dealt = 0;
    Zeros z = {};
    auto grid = [&]() {
        const int64_t mine = each < chunks - dealt ? each : chunks - dealt;
        z.p = static_cast<uint16_t*>(a.out) + dealt * ZERO_CHUNK;
        z.count = half_words - dealt * ZERO_CHUNK < mine * ZERO_CHUNK ? half_words - dealt * ZERO_CHUNK : mine * ZERO_CHUNK;
        dealt += mine;
        return dim3(static_cast<unsigned>(p.tiles + (mine < ZERO_GROUPS ? mine : ZERO_GROUPS)));
    };
    const uint2* in = nullptr;   // the ids themselves
    for (int pass = 0; pass < p.passes; ++pass) {
        uint2* out = (p.passes - pass) & 1 ? a.sorted : a.other;
        const dim3 counting = grid();
        hipLaunchKernelGGL(digit_counts, counting, dim3(SORT_BLOCK), 0, stream, a, z, in, pass * p.bits, p.bits);
        SPARC_CHECK_LAUNCH();
        const dim3 scattering = grid();
        hipLaunchKernelGGL(digit_scatter, scattering, dim3(SORT_BLOCK), lds, stream, a, z, in, out, pass * p.bits, p.bits);
        SPARC_CHECK_LAUNCH();
        in = out;
    }
    const size_t staged = static_cast<size_t>(p.per * p.in_group + 2 * MARGIN) * 2 * sizeof(uint32_t) +
                          (static_cast<size_t>(WAVES * VE) << p.lanes_log2) * sizeof(float);
    const bool once = a.n * a.dim * static_cast<int64_t>(sizeof(typename Elem<DT>::type)) > SPARC_KEEP_BYTES;
    hipLaunchKernelGGL((once ? row_sums<DT, VE, true> : row_sums<DT, VE, false>),
                       dim3(static_cast<unsigned>(ceil_div(p.workers, p.in_group)), static_cast<unsigned>(p.slices)), dim3(BLOCK), staged, stream,
                       a, p.lanes_log2);
    SPARC_CHECK_LAUNCH();
    const int slices = (a.dim + JOIN_COLS - 1) / JOIN_COLS, rows_at_once = 2048 / slices;
    const dim3 joining(static_cast<unsigned>(rows_at_once < 32 ? 32 : rows_at_once > 256 ? 256 : rows_at_once), static_cast<unsigned>(slices));
    if (a.dim >= 4) hipLaunchKernelGGL((join_rows<DT, 4>), joining, dim3(JOIN_THREADS), 0, stream, a);
    else hipLaunchKernelGGL((join_rows<DT, 1>), joining, dim3(JOIN_THREADS), 0, stream, a);
    SPARC_CHECK_LAUNCH();
    return SPARC_OK;
}

int launch_zeros(void* out, const int64_t bytes, sparc_stream_t stream) {
    const int64_t chunks = ceil_div(bytes / 2, ZERO_CHUNK);
    hipLaunchKernelGGL(zeros_kernel, dim3(static_cast<unsigned>(chunks < ZERO_GROUPS ? chunks : ZERO_GROUPS)), dim3(SORT_BLOCK), 0, stream,
                       (Zeros{static_cast<uint16_t*>(out), bytes / 2}));
    SPARC_CHECK_LAUNCH();
    return SPARC_OK;
}

template <int DT, int VE>
int launch_few(const GradArgs& a, sparc_stream_t stream) {
    int slices, blocks_log2 = FEW_BLOCKS_LOG2;
    const int lanes_log2 = lanes_for(ceil_div(a.dim, VE), &slices, FEW_LANES_LOG2);
    while (blocks_log2 > 4 && static_cast<int64_t>(slices) << blocks_log2 > 1 << FEW_BLOCKS_LOG2) --blocks_log2;   // two per CU in all
    Dealt d = {0, 0, 0};
    while ((static_cast<int64_t>(a.dim) * static_cast<int64_t>(sizeof(typename Elem<DT>::type)) << d.group) < GROUP_BYTES) ++d.group;
    const int64_t groups = ceil_div(a.rows, static_cast<int64_t>(1) << d.group);
    while (d.blocks < blocks_log2 && (static_cast<int64_t>(1) << d.blocks) < groups) ++d.blocks;
    // (a row's number inside its workgroup leaves a bit of the key for the one that pads the sort)
    while ((ceil_div(groups, static_cast<int64_t>(1) << d.blocks) << d.group) > (1 << (31 - PLACE_BITS))) ++d.blocks;
    while ((ceil_div(groups, static_cast<int64_t>(1) << d.blocks) << d.group) > (static_cast<int64_t>(1) << d.bits)) ++d.bits;
    const unsigned grid = static_cast<unsigned>(groups < (1 << d.blocks) ? groups : 1 << d.blocks);
    // Zeros that outgrow the Infinity Cache come in a launch of their own, line after line; where a workgroup's rows are not
    // whole lines of 128 bytes, from a third of that on, because lines that two workgroups write leave the cache half written.
    // Ten tokens, three outputs in turn, together and apart: 2449029 rows of 47 floats 173, 78 us; of 64 floats 115, 105;
    // 100000 of 507 halves 32, 22; of 512 halves 21.9, 22.9; 50000 of 507 halves 11.9, 12.7.
    const int64_t row_bytes = a.dim * static_cast<int64_t>(sizeof(typename Elem<DT>::type)), bytes = a.rows * row_bytes;
    const bool apart = bytes > ((row_bytes << d.group) % 128 ? SPARC_KEEP_BYTES / 3 : SPARC_KEEP_BYTES);
    if (apart) {
        const int rc = launch_zeros(a.out, bytes, stream);
        if (rc != SPARC_OK) return rc;
    }
    const size_t keys = (static_cast<size_t>(a.n) + 3) & ~static_cast<size_t>(3);
    hipLaunchKernelGGL((few_tokens<DT, VE>), dim3(grid, static_cast<unsigned>(slices)), dim3(FEW_THREADS), keys * sizeof(uint32_t), stream, a, d,
                       lanes_log2, !apart);
    SPARC_CHECK_LAUNCH();
    return SPARC_OK;
}

}  // namespace

extern "C" int sparc_embedding_grad(int64_t n, int64_t rows, int64_t dim, int dtype, const void* ids, int ids_64, const void* g,
                                    int64_t ldg, double scale, int64_t padding_idx, void* out, void* ws, size_t ws_bytes,
                                    sparc_stream_t stream) {
    if (n < 0 || rows < 0 || dim < 0 || dtype < SPARC_F32 || dtype > SPARC_F16 || ldg < dim || !out || (n > 0 && (!ids || !g)))
        return SPARC_ERR_ARG;
    if (n > SPARC_EMBEDDING_MAX || rows > SPARC_EMBEDDING_MAX || dim > SPARC_EMBEDDING_MAX_DIM) return SPARC_ERR_SIZE;
    if (rows == 0 || dim == 0) return SPARC_OK;
    if (n == 0) return launch_zeros(out, rows * dim * (dtype == SPARC_F32 ? 4 : 2), stream);   // (the sort would launch empty grids)
    const int ve = elements_of_16_bytes(dtype), used_ve = dim >= ve ? ve : 1;
    GradArgs a = {};
    Plan p = {};
    const bool few = few_enough(n, dim, dtype);
    if (!few) {
        p = plan_of(n, rows, static_cast<int>(dim), used_ve);
        bool ok;
        size_t used;
        a = carve(p, n, static_cast<int>(dim), ws, ws_bytes, &ok, &used);
        if (!ws || !ok) return SPARC_ERR_WS;
        a.per = p.per;
        while (1 << a.group_log2 < p.in_group) ++a.group_log2;
        a.long_row = p.long_row;
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
    a.dim = static_cast<int>(dim);
    a.wide_ids = ids_64 ? 1 : 0;
    a.scale = static_cast<float>(scale);
    return dispatch(dtype, dim, [&](auto type, auto width) {
        constexpr int DT = decltype(type)::value, VE = decltype(width)::value;
        return few ? launch_few<DT, VE>(a, stream) : launch_grad<DT, VE>(a, p, stream);
    });
}
