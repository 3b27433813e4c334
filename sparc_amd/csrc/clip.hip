// The global norm of many gradient tensors, clipping by it, and the Adam step that clips on the way.
//
//     N = sqrt(sum_t sum_j g_t[j]^2),   c = min(1, max_norm / (N + 1e-6)),   g_t <- round(c g_t)
//
// The squares are summed in float64: those of float32 gradients leave float32's range below 1e-19 and above 1e19, and
// the conversion is free behind the loads.  A pass over the gradients leaves one partial sum per workgroup (at most
// PARTS of them, in the grid's order); whoever needs the coefficient adds them up itself, every workgroup the same
// numbers in the same order, so there is neither a launch nor an arrival counter between the two passes and runs repeat
// bit for bit.  Short lists take one launch (clip_once_kernel, adam_once_kernel).
//
// Measured.  629 MB of float32 (a table and an MLP): norm 100 us = 6.3 TB/s, scaling 194 us = 6.5 TB/s; plain accesses:
// 161 and 204 us, because what the norm's pass leaves in the Infinity Cache is gone when the scaling comes to it, and what
// the scaling leaves there has to be written back under the next pass.  Without the last 192 MB that the norm's pass reads
// plainly for the scaling, which goes backwards: 94 and 205 us.  Lists below 192 MB stay plain: 160 MB, three lists in turn, 80 us
// streamed, 93 us plain; one list again and again 80 and 72 us.
// 6.4 MB (the MLP alone): 4.0 + 6.0 us, of which launches and the chain parts -> sum -> root -> quotient are most; the
// host's two launches and checks take longer (16.3 us a call).
// Adam on 31.5 M floats (883 MB): norm 24 us, update 136 us = 6.5 TB/s; plain accesses 40 and 160 us.  Below 192 MB plain:
// 8 M floats 49.1 us streamed, 49.7 us plain; 4 M 27.8 and 25.1.
#include <type_traits>

#include "adam.h"
#include "elem.h"
#include "ranges.h"

namespace {

constexpr int BLOCK = 256;
constexpr int BLOCK_BYTES = 16384;   // of one tensor per workgroup and turn: four 16-byte loads in flight per thread
constexpr int NORM_THREADS = 1024, NORM_BYTES = 65536;   // the same of the norm's pass, which has a partial sum per workgroup
constexpr int PARTS = 512;           // partial sums of one launch: two workgroups per CU
constexpr int MOST_BLOCKS = 65536;   // workgroups of a launch that writes
constexpr int ADAM_ELEMS = 1024;     // elements of one tensor per workgroup and turn of the Adam step
constexpr int ADAM_MOST = 64;        // tensors per launch of the Adam step
// What the 256 MB Infinity Cache is left to keep from one pass to the next.  Longer lists go by with streaming (nontemporal)
// accesses, but for their last KEEP_BYTES in the norm's pass, which the scaling, going backwards, finds there.
constexpr int64_t KEEP_BYTES = SPARC_KEEP_BYTES;

// Arguments of 2.5 KiB make a launch 0.9 us longer than some of 0.4 (4.1, 2.9 to 3.5 us): short lists have records for SHORT.
constexpr int SHORT = 16;

template <int R>
struct GradArgs {
    void* p[R];
    int64_t n_dtype[R];           // elements << 2 | type
    int32_t first_block[R];       // where tensor i's blocks begin; behind the last tensor: INT32_MAX
    int blocks, plain_from;                            // blocks from plain_from on are read without streaming
};

__device__ __forceinline__ int64_t lane_value(const int64_t v, const int lane) {
    const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(v), lane), hi = __builtin_amdgcn_readlane(static_cast<int>(v >> 32), lane);
    return static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo);
}

// The records of a launch, one or two per lane: a search for a block's tensor is two ballots and no load.
template <int R>
struct Records {
    static_assert(R <= 64 || R == 128, "one or two records per lane");
    static constexpr int H = R > 64 ? 2 : 1;
    int64_t p[H], n_dtype[H];
    int32_t first[H];
    __device__ __forceinline__ Records(const GradArgs<R>& a) {
        const int lane = threadIdx.x & 63, own = lane < R ? lane : 0;
#pragma unroll
        for (int h = 0; h < H; ++h) {
            p[h] = reinterpret_cast<int64_t>(a.p[own + 64 * h]);
            n_dtype[h] = a.n_dtype[own + 64 * h];
            first[h] = lane < R ? a.first_block[own + 64 * h] : INT32_MAX;
        }
    }
    // Block b: its tensor, elements and type, and which of the tensor's blocks it is (all uniform).
    __device__ __forceinline__ void find(const int b, void** base, int64_t* n, int* dtype, int64_t* k) const {
        int t = __popcll(__ballot(first[0] <= b)) - 1;
        if constexpr (H > 1) t += __popcll(__ballot(first[H - 1] <= b));
        const bool upper = H > 1 && t >= 64;
        const int lane = t & 63;
        *base = reinterpret_cast<void*>(lane_value(upper ? p[H - 1] : p[0], lane));
        const int64_t nd = lane_value(upper ? n_dtype[H - 1] : n_dtype[0], lane);
        *n = nd >> 2;
        *dtype = static_cast<int>(nd) & 3;
        *k = b - __builtin_amdgcn_readlane(upper ? first[H - 1] : first[0], lane);
    }
};

__device__ __forceinline__ double block_sum(double v, double* lds) {
    v = wave_sum(v);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    return lds[0] + lds[1] + lds[2] + lds[3];
}

template <int DT, bool STREAM>
__device__ __forceinline__ double squares(const void* p, const int64_t n, const int64_t k) {
    typedef typename Elem<DT>::type T;
    constexpr int VE = 16 / sizeof(T), TURNS = NORM_BYTES / (NORM_THREADS * 16);
    const int64_t e0 = k * (NORM_BYTES / static_cast<int>(sizeof(T)));
    const T* g = static_cast<const T*>(p) + e0 + threadIdx.x * VE;
    double s = 0.0;
    auto add = [&s](const Vec<DT, VE>& v) {
#pragma unroll
        for (int i = 0; i < VE; ++i) {
            const double x = v.get(i);
            s = fma(x, x, s);
        }
    };
    if (e0 + NORM_BYTES / static_cast<int>(sizeof(T)) <= n) {
        Vec<DT, VE> v[TURNS];
#pragma unroll
        for (int j = 0; j < TURNS; ++j) v[j].template load<STREAM>(g + j * NORM_THREADS * VE);
#pragma unroll
        for (int j = 0; j < TURNS; ++j) add(v[j]);
    } else {   // the tensor's end: whole vectors, all loads at once, and an element each for the first threads
        const int64_t here = n - e0, left = here - static_cast<int64_t>(threadIdx.x) * VE;
        const int rest = static_cast<int>(here % VE);
        const T* last = static_cast<const T*>(p) + n - rest;
        const double x = static_cast<int>(threadIdx.x) < rest ? Elem<DT>::up(last[threadIdx.x]) : 0.f;
        Vec<DT, VE> v[TURNS];
#pragma unroll
        for (int j = 0; j < TURNS; ++j)
            if (j * NORM_THREADS * VE + VE <= left) v[j].load(g + j * NORM_THREADS * VE);
#pragma unroll
        for (int j = 0; j < TURNS; ++j)
            if (j * NORM_THREADS * VE + VE <= left) add(v[j]);
        s = fma(x, x, s);
    }
    return s;
}

template <bool STREAM, int R>
__device__ __forceinline__ double squares_of_block(const Records<R>& records, const int b) {
    void* p;
    int64_t n, k;
    int dtype;
    records.find(b, &p, &n, &dtype, &k);
    return dtype == SPARC_F32 ? squares<SPARC_F32, STREAM>(p, n, k)
           : dtype == SPARC_BF16 ? squares<SPARC_BF16, STREAM>(p, n, k) : squares<SPARC_F16, STREAM>(p, n, k);
}

template <int R>
__global__ __launch_bounds__(NORM_THREADS, 8) void grad_squares_kernel(const GradArgs<R> a, double* parts) {
    __shared__ double lds[NORM_THREADS / 64];
    const Records<R> records(a);
    double s = 0.0;
    int b = blockIdx.x;
    for (; b < a.plain_from; b += gridDim.x) s += squares_of_block<true>(records, b);
    for (; b < a.blocks; b += gridDim.x) s += squares_of_block<false>(records, b);
    s = wave_sum(s);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        s = lds[0];
        for (int w = 1; w < NORM_THREADS / 64; ++w) s += lds[w];
        parts[blockIdx.x] = s;
    }
}

// parts[0] = the sum of parts[0 .. n): for lists that took more than one launch.
__global__ __launch_bounds__(BLOCK) void grad_parts_kernel(double* parts, const int64_t n) {
    __shared__ double lds[BLOCK / 64];
    double s = 0.0;
    for (int64_t i = threadIdx.x; i < n; i += BLOCK) s += parts[i];
    s = block_sum(s, lds);
    if (threadIdx.x == 0) parts[0] = s;
}

struct Clip {
    const double* parts;
    float* norm_out;   // null: another launch of the same call writes it
    double max_norm;
    int n_parts;
};

// A norm that is not finite gives what the formula gives: 0 for an infinite one (so infinite gradients become NaN), NaN for
// NaN; an infinite max_norm never clips.
__device__ __forceinline__ float coefficient_of(const double norm, const double max_norm) {
    const double coef = isinf(max_norm) ? 1.0 : max_norm / (norm + 1e-6);
    return coef >= 1.0 ? 1.f : static_cast<float>(coef);
}

// The coefficient, in every thread: the partial sums are requested first of all, and added up where the coefficient is first
// asked for, behind the loads that do not need it.
struct Coefficient {
    const Clip& c;
    double* lds;
    double parts;
    float value;
    bool known;
    __device__ __forceinline__ Coefficient(const Clip& clip, double* scratch) : c(clip), lds(scratch), parts(0.0), value(0.f), known(false) {
        static_assert(PARTS <= 2 * BLOCK, "two partial sums per thread");
        const int i = threadIdx.x;
        const double first = i < c.n_parts ? c.parts[i] : 0.0, second = i + BLOCK < c.n_parts ? c.parts[i + BLOCK] : 0.0;
        parts = first + second;
    }
    __device__ __forceinline__ float get() {   // by the whole workgroup
        if (!known) {
            const double norm = sqrt(block_sum(parts, lds));
            if (c.norm_out && blockIdx.x == 0 && threadIdx.x == 0) *c.norm_out = static_cast<float>(norm);
            value = coefficient_of(norm, c.max_norm);
            known = true;
        }
        return value;
    }
};

template <int DT, bool STREAM>
__device__ __forceinline__ void scale_block(void* p, const int64_t n, const int64_t k, Coefficient& c) {
    typedef typename Elem<DT>::type T;
    constexpr int VE = 16 / sizeof(T), TURNS = BLOCK_BYTES / (BLOCK * 16);
    const int64_t e0 = k * (BLOCK_BYTES / static_cast<int>(sizeof(T)));
    T* g = static_cast<T*>(p) + e0 + threadIdx.x * VE;
    auto scaled = [](Vec<DT, VE>& v, const float coef) {
#pragma unroll
        for (int i = 0; i < VE; ++i) v.set(i, v.get(i) * coef);
    };
    if (e0 + BLOCK_BYTES / static_cast<int>(sizeof(T)) <= n) {
        Vec<DT, VE> v[TURNS];
#pragma unroll
        for (int j = 0; j < TURNS; ++j) v[j].template load<STREAM>(g + j * BLOCK * VE);
        const float coef = c.get();
#pragma unroll
        for (int j = 0; j < TURNS; ++j) {
            scaled(v[j], coef);
            v[j].template store<STREAM>(g + j * BLOCK * VE);
        }
    } else {   // the tensor's end: whole vectors, all loads at once, and an element each for the first threads
        const int64_t here = n - e0, left = here - static_cast<int64_t>(threadIdx.x) * VE;
        const int rest = static_cast<int>(here % VE);
        T* last = static_cast<T*>(p) + n - rest;
        const float x = static_cast<int>(threadIdx.x) < rest ? Elem<DT>::up(last[threadIdx.x]) : 0.f;
        Vec<DT, VE> v[TURNS];
#pragma unroll
        for (int j = 0; j < TURNS; ++j)
            if (j * BLOCK * VE + VE <= left) v[j].load(g + j * BLOCK * VE);
        const float coef = c.get();
#pragma unroll
        for (int j = 0; j < TURNS; ++j)
            if (j * BLOCK * VE + VE <= left) {
                scaled(v[j], coef);
                v[j].store(g + j * BLOCK * VE);
            }
        if (static_cast<int>(threadIdx.x) < rest) last[threadIdx.x] = Elem<DT>::down(x * coef);
    }
}

// From the last block to the first: the norm's pass left the last ones in the cache.
template <bool STREAM, int R>
__global__ __launch_bounds__(BLOCK) void grad_scale_kernel(const GradArgs<R> a, const Clip clip) {
    __shared__ double lds[BLOCK / 64];
    Coefficient c(clip, lds);
    const Records<R> records(a);
    for (int b = a.blocks - 1 - static_cast<int>(blockIdx.x); b >= 0; b -= gridDim.x) {
        void* p;
        int64_t n, k;
        int dtype;
        records.find(b, &p, &n, &dtype, &k);
        if (dtype == SPARC_F32) scale_block<SPARC_F32, STREAM>(p, n, k, c);
        else if (dtype == SPARC_BF16) scale_block<SPARC_BF16, STREAM>(p, n, k, c);
        else scale_block<SPARC_F16, STREAM>(p, n, k, c);
    }
    c.get();   // (a list without elements has a norm too)
}

template <int R>
struct AdamClipArgs {
    sparc_adam_tensor_t t[R];
    int32_t first_block[R];   // where tensor i's blocks begin; behind the last tensor: INT32_MAX
    int blocks;
    AdamFactors by;
};

template <bool STREAM, int R>
__global__ __launch_bounds__(BLOCK) void adam_clip_kernel(const AdamClipArgs<R> a, const Clip clip) {
    __shared__ double lds[BLOCK / 64];
    typedef Vec<SPARC_F32, 4> V4;
    Coefficient c(clip, lds);
    const int lane = threadIdx.x & 63;
    const sparc_adam_tensor_t mine = a.t[lane < R ? lane : 0];
    const int32_t first = lane < R ? a.first_block[lane < R ? lane : 0] : INT32_MAX;
    static_assert(R <= 64, "a record per lane");
    for (int b = blockIdx.x; b < a.blocks; b += gridDim.x) {
        const int of = __popcll(__ballot(first <= b)) - 1;
        float* tp = reinterpret_cast<float*>(lane_value(reinterpret_cast<int64_t>(mine.p), of));
        const float* tg = reinterpret_cast<const float*>(lane_value(reinterpret_cast<int64_t>(mine.g), of));
        float* tm = reinterpret_cast<float*>(lane_value(reinterpret_cast<int64_t>(mine.m), of));
        float* tv = reinterpret_cast<float*>(lane_value(reinterpret_cast<int64_t>(mine.v), of));
        const int64_t n = lane_value(mine.n, of);
        const int64_t e = static_cast<int64_t>(b - __builtin_amdgcn_readlane(first, of)) * ADAM_ELEMS + threadIdx.x * 4;
        const bool whole = e + 4 <= n;
        V4 p = {}, g = {}, m = {}, v = {};
        if (whole) {
            g.load<STREAM>(tg + e);
            p.load<STREAM>(tp + e);
            m.load<STREAM>(tm + e);
            v.load<STREAM>(tv + e);
        } else {   // the tensor's end
#pragma unroll
            for (int i = 0; i < 3; ++i)
                if (e + i < n) {
                    g.v[i] = tg[e + i];
                    p.v[i] = tp[e + i];
                    m.v[i] = tm[e + i];
                    v.v[i] = tv[e + i];
                }
        }
        const float coef = c.get();
        if (e >= n) continue;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float pi = p.v[i], mi = m.v[i], vi = v.v[i];
            adam_one(pi, g.v[i], mi, vi, a.by, coef);
            p.v[i] = pi; m.v[i] = mi; v.v[i] = vi;
        }
        if (whole) {
            p.store<STREAM>(tp + e);
            m.store<STREAM>(tm + e);
            v.store<STREAM>(tv + e);
        } else {
#pragma unroll
            for (int i = 0; i < 3; ++i)
                if (e + i < n) {
                    tp[e + i] = p.v[i];
                    tm[e + i] = m.v[i];
                    tv[e + i] = v.v[i];
                }
        }
    }
    c.get();   // (a list without elements has a norm too)
}

// ---- short lists in one launch ----------------------------------------------------------------------------

// One workgroup holds the whole list in registers: squares, their sum, the coefficient, and back.  A launch less, of the two
// that a call with little data mostly consists of.  Blocks of a tensor go to the waves in turn.  A call among others and one
// that is waited for, two launches and one: clipping 6000 floats 13.8, 23.6 us and 10.4, 20.6; 128 KiB of bfloat16 13.6, 23.8
// and 10.0, 24.0; 256 KiB 13.7, 24.0 and 11.6, 27.7, hence the limit of 128.  Adam on 6000 parameters 15.0, 25.0 and 11.5, 22.6;
// on 16384 14.8, 24.9 and 11.0, 26.2.
constexpr int ONCE_WAVES = 16, ONCE_THREADS = 64 * ONCE_WAVES, ONCE_TURNS = 4, ONCE_BLOCKS = ONCE_WAVES * ONCE_TURNS;
constexpr int ONCE_VECTORS = 2, ONCE_BYTES = 64 * 16 * ONCE_VECTORS;   // of a block of the clipping
constexpr int ONCE_ELEMS = 64 * 4;                                     // of a block of the Adam step
typedef uint32_t Raw __attribute__((ext_vector_type(4)));              // 16 bytes of a gradient, whatever the type

template <int DT>
struct OnceBlock {
    typedef typename Elem<DT>::type T;
    static constexpr int VE = 16 / sizeof(T);
    typedef Vec<DT, VE> V;
    T* g;
    int64_t left;   // elements from this lane's first on
    __device__ __forceinline__ OnceBlock(void* p, const int64_t n, const int64_t k) {
        const int64_t e = k * (ONCE_BYTES / static_cast<int>(sizeof(T))) + (threadIdx.x & 63) * VE;
        g = static_cast<T*>(p) + e;
        left = n - e;
    }
    __device__ __forceinline__ void load(Raw* r) const {
#pragma unroll
        for (int j = 0; j < ONCE_VECTORS; ++j) {
            V v;
            const int64_t here = left - j * 64 * VE;
            if (here >= VE) v.load(g + j * 64 * VE);
            else {   // the tensor's end
#pragma unroll
                for (int c = 0; c < VE; ++c) v.v[c] = c < here ? g[j * 64 * VE + c] : Elem<DT>::down(0.f);
            }
            r[j] = __builtin_bit_cast(Raw, v);
        }
    }
    static __device__ __forceinline__ double squares(const Raw* r) {
        double s = 0.0;
#pragma unroll
        for (int j = 0; j < ONCE_VECTORS; ++j) {
            const V v = __builtin_bit_cast(V, r[j]);
#pragma unroll
            for (int c = 0; c < VE; ++c) {
                const double x = v.get(c);
                s = fma(x, x, s);
            }
        }
        return s;
    }
    __device__ __forceinline__ void store(const Raw* r, const float coef) const {
#pragma unroll
        for (int j = 0; j < ONCE_VECTORS; ++j) {
            V v = __builtin_bit_cast(V, r[j]);
#pragma unroll
            for (int c = 0; c < VE; ++c) v.set(c, v.get(c) * coef);
            const int64_t here = left - j * 64 * VE;
            if (here >= VE) v.store(g + j * 64 * VE);
            else {
#pragma unroll
                for (int c = 0; c < VE; ++c)
                    if (c < here) g[j * 64 * VE + c] = v.v[c];
            }
        }
    }
};

// The coefficient of the workgroup's sum of squares; the norm goes to *norm_out.
__device__ __forceinline__ float once_coefficient(double s, double* lds, const double max_norm, float* norm_out) {
    s = wave_sum(s);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = s;
    __syncthreads();
    s = lds[0];
#pragma unroll
    for (int w = 1; w < ONCE_WAVES; ++w) s += lds[w];
    const double norm = sqrt(s);
    if (threadIdx.x == 0) *norm_out = static_cast<float>(norm);
    return coefficient_of(norm, max_norm);
}

template <int R>
__global__ __launch_bounds__(ONCE_THREADS) void clip_once_kernel(const GradArgs<R> a, const double max_norm, float* norm_out) {
    __shared__ double lds[ONCE_WAVES];
    const Records<R> records(a);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Raw r[ONCE_TURNS][ONCE_VECTORS];
    auto each = [&](auto&& f) {
#pragma unroll
        for (int t = 0; t < ONCE_TURNS; ++t) {
            const int b = wave + t * ONCE_WAVES;
            if (b >= a.blocks) break;
            void* p;
            int64_t n, k;
            int dtype;
            records.find(b, &p, &n, &dtype, &k);
            if (dtype == SPARC_F32) f(OnceBlock<SPARC_F32>(p, n, k), r[t]);
            else if (dtype == SPARC_BF16) f(OnceBlock<SPARC_BF16>(p, n, k), r[t]);
            else f(OnceBlock<SPARC_F16>(p, n, k), r[t]);
        }
    };
    each([](const auto& block, Raw* v) { block.load(v); });
    double s = 0.0;
    each([&s](const auto& block, Raw* v) { s += block.squares(v); });
    const float coef = once_coefficient(s, lds, max_norm, norm_out);
    each([coef](const auto& block, Raw* v) { block.store(v, coef); });
}

template <int R>
__global__ __launch_bounds__(ONCE_THREADS) void adam_once_kernel(const AdamClipArgs<R> a, const double max_norm, float* norm_out) {
    __shared__ double lds[ONCE_WAVES];
    typedef Vec<SPARC_F32, 4> V4;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const sparc_adam_tensor_t mine = a.t[lane < R ? lane : 0];
    const int32_t first = lane < R ? a.first_block[lane < R ? lane : 0] : INT32_MAX;
    V4 p[ONCE_TURNS] = {}, g[ONCE_TURNS] = {}, m[ONCE_TURNS] = {}, v[ONCE_TURNS] = {};
    float *tp[ONCE_TURNS], *tm[ONCE_TURNS], *tv[ONCE_TURNS];
    int64_t left[ONCE_TURNS];
    double s = 0.0;
#pragma unroll
    for (int t = 0; t < ONCE_TURNS; ++t) {
        const int b = wave + t * ONCE_WAVES;
        if (b >= a.blocks) break;
        const int of = __popcll(__ballot(first <= b)) - 1;
        const int64_t e = static_cast<int64_t>(b - __builtin_amdgcn_readlane(first, of)) * ONCE_ELEMS + lane * 4;
        left[t] = lane_value(mine.n, of) - e;
        const float* tg = reinterpret_cast<const float*>(lane_value(reinterpret_cast<int64_t>(mine.g), of)) + e;
        tp[t] = reinterpret_cast<float*>(lane_value(reinterpret_cast<int64_t>(mine.p), of)) + e;
        tm[t] = reinterpret_cast<float*>(lane_value(reinterpret_cast<int64_t>(mine.m), of)) + e;
        tv[t] = reinterpret_cast<float*>(lane_value(reinterpret_cast<int64_t>(mine.v), of)) + e;
        if (left[t] >= 4) {
            g[t].load(tg);
            p[t].load(tp[t]);
            m[t].load(tm[t]);
            v[t].load(tv[t]);
        } else {
#pragma unroll
            for (int i = 0; i < 3; ++i)
                if (i < left[t]) {
                    g[t].v[i] = tg[i];
                    p[t].v[i] = tp[t][i];
                    m[t].v[i] = tm[t][i];
                    v[t].v[i] = tv[t][i];
                }
        }
    }
#pragma unroll
    for (int t = 0; t < ONCE_TURNS; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const double x = g[t].v[i];
            s = fma(x, x, s);
        }
    const float coef = once_coefficient(s, lds, max_norm, norm_out);
#pragma unroll
    for (int t = 0; t < ONCE_TURNS; ++t) {
        if (wave + t * ONCE_WAVES >= a.blocks) break;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float pi = p[t].v[i], mi = m[t].v[i], vi = v[t].v[i];
            adam_one(pi, g[t].v[i], mi, vi, a.by, coef);
            p[t].v[i] = pi; m[t].v[i] = mi; v[t].v[i] = vi;
        }
        if (left[t] >= 4) {
            p[t].store(tp[t]);
            m[t].store(tm[t]);
            v[t].store(tv[t]);
        } else {
#pragma unroll
            for (int i = 0; i < 3; ++i)
                if (i < left[t]) {
                    tp[t][i] = p[t].v[i];
                    tm[t][i] = m[t].v[i];
                    tv[t][i] = v[t].v[i];
                }
        }
    }
}

bool grads_ok(const int64_t n_tensors, const sparc_grad_tensor_t* t) {
    if (n_tensors < 0 || (n_tensors > 0 && !t)) return false;
    for (int64_t i = 0; i < n_tensors; ++i)
        if (t[i].n < 0 || t[i].n > SPARC_GRAD_MAX_ELEMS || (t[i].n > 0 && !t[i].p) || t[i].dtype < SPARC_F32 || t[i].dtype > SPARC_F16) return false;
    return true;
}

int64_t bytes_of(const sparc_grad_tensor_t& t) { return t.n * (t.dtype == SPARC_F32 ? 4 : 2); }

// The `count` tensors t(from), t(from + 1) ... as kernel arguments.  Their number of blocks stays below 2^30
// (SPARC_GRAD_MAX_ELEMS).  left: bytes of the list from there on.  Returns these tensors' bytes.
template <int R, typename F>
int64_t fill(GradArgs<R>& a, F&& t, const int64_t from, const int count, const int block_bytes, const int64_t left) {
    int64_t blocks = 0, bytes = 0;
    for (int i = 0; i < R; ++i) {
        const sparc_grad_tensor_t r = i < count ? t(from + i) : sparc_grad_tensor_t{nullptr, 0, 0};
        a.p[i] = r.p;
        a.n_dtype[i] = r.n << 2 | r.dtype;
        a.first_block[i] = i < count ? static_cast<int32_t>(blocks) : INT32_MAX;
        bytes += bytes_of(r);
        blocks += (bytes_of(r) + block_bytes - 1) / block_bytes;
    }
    a.blocks = static_cast<int>(blocks);
    const int64_t keep = KEEP_BYTES - (left - bytes);   // of these tensors' bytes
    const int64_t plain = keep <= 0 ? 0 : keep / block_bytes;
    a.plain_from = static_cast<int>(keep >= bytes || plain >= blocks ? 0 : blocks - plain);
    return bytes;
}

// f(the records of a launch that `count` of at most MOST tensors take, as an integral constant).
template <int MOST, typename F>
int with_records(const int64_t count, F&& f) {
    if (count <= SHORT) return f(std::integral_constant<int, SHORT>());
    return f(std::integral_constant<int, MOST>());
}

size_t parts_bytes_of(const int64_t n_tensors) {
    const int64_t launches = (n_tensors + SPARC_GRAD_MAX_TENSORS - 1) / SPARC_GRAD_MAX_TENSORS;
    return static_cast<size_t>(launches > 0 ? launches : 1) * PARTS * sizeof(double);
}

bool parts_ok(const int64_t n_tensors, const double* parts, const size_t bytes) {
    return bytes >= parts_bytes_of(n_tensors) && (reinterpret_cast<uintptr_t>(parts) & 7) == 0;
}

// The partial sums of the tensors t(0) ... t(n_tensors - 1), checked by the caller.
template <typename F>
int launch_norm(const int64_t n_tensors, F&& t, double* parts, const size_t parts_bytes, int64_t* n_parts, sparc_stream_t stream) {
    if (!parts_ok(n_tensors, parts, parts_bytes)) return SPARC_ERR_WS;
    int64_t total = 0, left = 0;
    int launches = 0;
    for (int64_t i = 0; i < n_tensors; ++i) left += bytes_of(t(i));
    for (int64_t from = 0; from < n_tensors; from += SPARC_GRAD_MAX_TENSORS) {
        const int count = static_cast<int>(n_tensors - from < SPARC_GRAD_MAX_TENSORS ? n_tensors - from : SPARC_GRAD_MAX_TENSORS);
        const int rc = with_records<SPARC_GRAD_MAX_TENSORS>(count, [&](auto records) {
            constexpr int R = decltype(records)::value;
            GradArgs<R> a;
            left -= fill(a, t, from, count, NORM_BYTES, left);
            if (a.blocks == 0) return SPARC_OK;
            const int grid = a.blocks < PARTS ? a.blocks : PARTS;
            hipLaunchKernelGGL((grad_squares_kernel<R>), dim3(grid), dim3(NORM_THREADS), 0, stream, a, parts + total);
            SPARC_CHECK_LAUNCH();
            total += grid;
            ++launches;
            return SPARC_OK;
        });
        if (rc != SPARC_OK) return rc;
    }
    if (launches > 1) {
        hipLaunchKernelGGL(grad_parts_kernel, dim3(1), dim3(BLOCK), 0, stream, parts, total);
        SPARC_CHECK_LAUNCH();
        total = 1;
    }
    *n_parts = total;
    return SPARC_OK;
}

struct AdamRates {
    double lr, beta1, beta2, eps, weight_decay;
    int64_t step;
};

bool adam_ok(const int64_t n_tensors, const sparc_adam_tensor_t* t, const AdamRates& r) {
    if (n_tensors < 0 || (n_tensors > 0 && !t) || r.step < 1 || !(r.beta1 >= 0.0 && r.beta1 < 1.0) || !(r.beta2 >= 0.0 && r.beta2 < 1.0) ||
        !(r.eps >= 0.0))
        return false;
    for (int64_t i = 0; i < n_tensors; ++i)
        if (t[i].n < 0 || t[i].n > SPARC_GRAD_MAX_ELEMS || (t[i].n > 0 && (!t[i].p || !t[i].g || !t[i].m || !t[i].v))) return false;
    return true;
}

// The first R of the n tensors t as kernel arguments, in fewer than 2^30 blocks.
template <int R>
void fill(AdamClipArgs<R>& a, const sparc_adam_tensor_t* t, const int64_t n, const AdamRates& r, const int block_elems) {
    int64_t blocks = 0;
    for (int i = 0; i < R; ++i) {
        a.t[i] = i < n ? t[i] : sparc_adam_tensor_t{};
        a.first_block[i] = i < n ? static_cast<int32_t>(blocks) : INT32_MAX;
        blocks += (a.t[i].n + block_elems - 1) / block_elems;
    }
    a.blocks = static_cast<int>(blocks);
    a.by = adam_factors(r.lr, r.beta1, r.beta2, r.eps, r.weight_decay, r.step);
}

int launch_adam(const int64_t n_tensors, const sparc_adam_tensor_t* tensors, const AdamRates& r, Clip c, sparc_stream_t stream) {
    int64_t all = 0;
    for (int64_t i = 0; i < n_tensors; ++i) all += tensors[i].n;
    for (int64_t from = 0; from < n_tensors || from == 0; from += ADAM_MOST) {
        const int rc = with_records<ADAM_MOST>(n_tensors - from, [&](auto records) {
            constexpr int R = decltype(records)::value;
            AdamClipArgs<R> a;
            fill(a, tensors + from, n_tensors - from, r, ADAM_ELEMS);
            if (a.blocks == 0 && !c.norm_out) return SPARC_OK;
            const int grid = a.blocks < 1 ? 1 : a.blocks < MOST_BLOCKS ? a.blocks : MOST_BLOCKS;
            if (16 * all > KEEP_BYTES) hipLaunchKernelGGL((adam_clip_kernel<true, R>), dim3(grid), dim3(BLOCK), 0, stream, a, c);
            else hipLaunchKernelGGL((adam_clip_kernel<false, R>), dim3(grid), dim3(BLOCK), 0, stream, a, c);
            SPARC_CHECK_LAUNCH();
            c.norm_out = nullptr;
            return SPARC_OK;
        });
        if (rc != SPARC_OK) return rc;
    }
    return SPARC_OK;
}

}  // namespace

extern "C" size_t sparc_grad_norm_workspace_bytes(int64_t n_tensors) { return n_tensors < 0 ? 0 : parts_bytes_of(n_tensors); }

extern "C" int sparc_grad_norm(int64_t n_tensors, const sparc_grad_tensor_t* tensors, double* parts, size_t parts_bytes,
                               int64_t* n_parts, sparc_stream_t stream) {
    if (!parts || !n_parts || !grads_ok(n_tensors, tensors)) return SPARC_ERR_ARG;
    return launch_norm(n_tensors, [&](int64_t i) { return tensors[i]; }, parts, parts_bytes, n_parts, stream);
}

extern "C" int sparc_clip_grad_norm(int64_t n_tensors, const sparc_grad_tensor_t* tensors, double max_norm, double* parts,
                                    size_t parts_bytes, float* norm_out, sparc_stream_t stream) {
    if (!norm_out || !(max_norm >= 0.0) || !parts || !grads_ok(n_tensors, tensors)) return SPARC_ERR_ARG;
    if (!parts_ok(n_tensors, parts, parts_bytes)) return SPARC_ERR_WS;
    const int apart = check_ranges(n_tensors, [tensors](const int64_t i) {
        const uintptr_t from = reinterpret_cast<uintptr_t>(tensors[i].p);
        return MemoryRange{from, from + bytes_of(tensors[i]), true};
    });
    if (apart != SPARC_OK) return apart;
    int64_t once = 0;
    for (int64_t i = 0; i < n_tensors && once <= ONCE_BLOCKS; ++i) once += (bytes_of(tensors[i]) + ONCE_BYTES - 1) / ONCE_BYTES;
    if (n_tensors <= SPARC_GRAD_MAX_TENSORS && once <= ONCE_BLOCKS) {
        return with_records<SPARC_GRAD_MAX_TENSORS>(n_tensors, [&](auto records) {
            constexpr int R = decltype(records)::value;
            GradArgs<R> a;
            fill(a, [&](int64_t k) { return tensors[k]; }, 0, static_cast<int>(n_tensors), ONCE_BYTES, 0);
            hipLaunchKernelGGL((clip_once_kernel<R>), dim3(1), dim3(ONCE_THREADS), 0, stream, a, max_norm, norm_out);
            SPARC_CHECK_LAUNCH();
            return SPARC_OK;
        });
    }
    int64_t n_parts = 0;
    const int rc = sparc_grad_norm(n_tensors, tensors, parts, parts_bytes, &n_parts, stream);
    if (rc != SPARC_OK) return rc;
    Clip c = {parts, norm_out, max_norm, static_cast<int>(n_parts)};
    int64_t left = 0;
    const int64_t launches = n_tensors ? (n_tensors + SPARC_GRAD_MAX_TENSORS - 1) / SPARC_GRAD_MAX_TENSORS : 1;
    for (int64_t i = launches - 1; i >= 0; --i) {   // backwards, as inside a launch
        const int64_t from = i * SPARC_GRAD_MAX_TENSORS;
        const int count = static_cast<int>(n_tensors - from < SPARC_GRAD_MAX_TENSORS ? n_tensors - from : SPARC_GRAD_MAX_TENSORS);
        for (int k = 0; k < count; ++k) left += bytes_of(tensors[from + k]);
        const int rc = with_records<SPARC_GRAD_MAX_TENSORS>(count, [&](auto records) {
            constexpr int R = decltype(records)::value;
            GradArgs<R> a;
            fill(a, [&](int64_t k) { return tensors[k]; }, from, count, BLOCK_BYTES, left);
            if (a.blocks == 0 && !c.norm_out) return SPARC_OK;
            const int grid = a.blocks < 1 ? 1 : a.blocks < MOST_BLOCKS ? a.blocks : MOST_BLOCKS;
            if (a.plain_from > 0) hipLaunchKernelGGL((grad_scale_kernel<true, R>), dim3(grid), dim3(BLOCK), 0, stream, a, c);
            else hipLaunchKernelGGL((grad_scale_kernel<false, R>), dim3(grid), dim3(BLOCK), 0, stream, a, c);
            SPARC_CHECK_LAUNCH();
            c.norm_out = nullptr;
            return SPARC_OK;
        });
        if (rc != SPARC_OK) return rc;
    }
    return SPARC_OK;
}

extern "C" int sparc_adam_step_clipped(int64_t n_tensors, const sparc_adam_tensor_t* tensors, double lr, double beta1, double beta2,
                                       double eps, double weight_decay, int64_t step, const double* parts, int64_t n_parts,
                                       double max_norm, float* norm_out, sparc_stream_t stream) {
    const AdamRates rates = {lr, beta1, beta2, eps, weight_decay, step};
    if (!adam_ok(n_tensors, tensors, rates) || !parts || !norm_out || n_parts < 0 || n_parts > PARTS || !(max_norm >= 0.0)) return SPARC_ERR_ARG;
    const int apart = check_adam_ranges(n_tensors, tensors);
    if (apart != SPARC_OK) return apart;
    return launch_adam(n_tensors, tensors, rates, Clip{parts, norm_out, max_norm, static_cast<int>(n_parts)}, stream);
}

extern "C" int sparc_clip_adam_step(int64_t n_tensors, const sparc_adam_tensor_t* tensors, double lr, double beta1, double beta2,
                                    double eps, double weight_decay, int64_t step, double max_norm, double* parts,
                                    size_t parts_bytes, float* norm_out, sparc_stream_t stream) {
    const AdamRates rates = {lr, beta1, beta2, eps, weight_decay, step};
    if (!adam_ok(n_tensors, tensors, rates) || !parts || !norm_out || !(max_norm >= 0.0)) return SPARC_ERR_ARG;
    if (!parts_ok(n_tensors, parts, parts_bytes)) return SPARC_ERR_WS;
    const int apart = check_adam_ranges(n_tensors, tensors);
    if (apart != SPARC_OK) return apart;
    int64_t once = 0;
    for (int64_t i = 0; i < n_tensors && once <= ONCE_BLOCKS; ++i) once += (tensors[i].n + ONCE_ELEMS - 1) / ONCE_ELEMS;
    if (n_tensors <= ADAM_MOST && once <= ONCE_BLOCKS) {
        return with_records<ADAM_MOST>(n_tensors, [&](auto records) {
            constexpr int R = decltype(records)::value;
            AdamClipArgs<R> a;
            fill(a, tensors, n_tensors, rates, ONCE_ELEMS);
            hipLaunchKernelGGL((adam_once_kernel<R>), dim3(1), dim3(ONCE_THREADS), 0, stream, a, max_norm, norm_out);
            SPARC_CHECK_LAUNCH();
            return SPARC_OK;
        });
    }
    int64_t n_parts = 0;
    auto gradient = [&](int64_t i) { return sparc_grad_tensor_t{const_cast<float*>(tensors[i].g), tensors[i].n, SPARC_F32}; };
    const int rc = launch_norm(n_tensors, gradient, parts, parts_bytes, &n_parts, stream);
    if (rc != SPARC_OK) return rc;
    return launch_adam(n_tensors, tensors, rates, Clip{parts, norm_out, max_norm, static_cast<int>(n_parts)}, stream);
}
