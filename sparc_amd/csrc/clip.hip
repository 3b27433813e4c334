// The global norm of many gradient tensors, clipping by it, and the Adam step that clips on the way.
//
//     N = sqrt(sum_t sum_j g_t[j]^2),   c = min(1, max_norm / (N + 1e-6)),   g_t <- round(c g_t)
//
// The squares are summed in float64: those of float32 gradients leave float32's range below 1e-19 and above 1e19, and
// the conversion is free behind the loads.  A pass over the gradients leaves one partial sum per workgroup (at most
// PARTS of them, in the grid's order); whoever needs the coefficient adds them up itself, every workgroup the same
// numbers in the same order, so there is neither a launch nor an arrival counter between the two passes and runs repeat
// bit for bit.
#include "elem.h"

namespace {

constexpr int BLOCK = 256;
constexpr int BLOCK_BYTES = 16384;   // of one tensor per workgroup and turn: four 16-byte loads in flight per thread
constexpr int NORM_THREADS = 1024, NORM_BYTES = 65536;   // the same of the norm's pass, which has a partial sum per workgroup
constexpr int PARTS = 512;           // partial sums of one launch: two workgroups per CU
constexpr int MOST_BLOCKS = 2048;    // workgroups of a launch that writes: eight per CU
constexpr int ADAM_ELEMS = 1024;     // elements of one tensor per workgroup and turn of the Adam step
constexpr int ADAM_MOST = 48;        // tensors per launch of the Adam step

struct GradArgs {
    void* p[SPARC_GRAD_MAX_TENSORS];
    int64_t n[SPARC_GRAD_MAX_TENSORS];
    int32_t first_block[SPARC_GRAD_MAX_TENSORS + 1];   // blocks [first_block[i], first_block[i + 1]) belong to tensor i
    uint8_t dtype[SPARC_GRAD_MAX_TENSORS];
    int n_tensors;
};

// Index of the tensor that block b belongs to (wave-uniform; tensors without elements own no block).
template <class A>
__device__ __forceinline__ int tensor_of(const A& a, const int b) {
    int lo = 0, hi = a.n_tensors;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.first_block[mid] <= b) lo = mid;
        else hi = mid;
    }
    return lo;
}

__device__ __forceinline__ double block_sum(double v, double* lds) {
    v = wave_sum(v);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    return lds[0] + lds[1] + lds[2] + lds[3];
}

template <int DT>
__device__ __forceinline__ double squares(const void* p, const int64_t n, const int64_t e0) {
    typedef typename Elem<DT>::type T;
    constexpr int VE = 16 / sizeof(T), TURNS = NORM_BYTES / (NORM_THREADS * 16);
    const T* g = static_cast<const T*>(p);
    double s = 0.0;
    Vec<DT, VE> v[TURNS];
#pragma unroll
    for (int k = 0; k < TURNS; ++k) {
        const int64_t e = e0 + (k * NORM_THREADS + threadIdx.x) * VE;
        if (e + VE <= n) {
            v[k].load(g + e);
        } else {   // the tensor's last vector, and behind it
#pragma unroll
            for (int i = 0; i < VE; ++i) v[k].set(i, e + i < n ? Elem<DT>::up(g[e + i]) : 0.f);
        }
    }
#pragma unroll
    for (int k = 0; k < TURNS; ++k)
#pragma unroll
        for (int i = 0; i < VE; ++i) {
            const double x = v[k].get(i);
            s = fma(x, x, s);
        }
    return s;
}

__global__ __launch_bounds__(NORM_THREADS) void grad_squares_kernel(const GradArgs a, const int blocks, double* parts) {
    __shared__ double lds[NORM_THREADS / 64];
    double s = 0.0;
    for (int b = blockIdx.x; b < blocks; b += gridDim.x) {
        const int t = tensor_of(a, b);
        const int64_t k = b - a.first_block[t];
        if (a.dtype[t] == SPARC_F32) s += squares<SPARC_F32>(a.p[t], a.n[t], k * (NORM_BYTES / 4));
        else if (a.dtype[t] == SPARC_BF16) s += squares<SPARC_BF16>(a.p[t], a.n[t], k * (NORM_BYTES / 2));
        else s += squares<SPARC_F16>(a.p[t], a.n[t], k * (NORM_BYTES / 2));
    }
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

// The coefficient, in every thread.  A norm that is not finite gives what the formula gives: 0 for an infinite one (so
// infinite gradients become NaN), NaN for NaN; an infinite max_norm never clips.
__device__ __forceinline__ float clip_coef(const Clip& c, double* lds) {
    double s = 0.0;
    for (int i = threadIdx.x; i < c.n_parts; i += BLOCK) s += c.parts[i];
    s = block_sum(s, lds);
    const double norm = sqrt(s);
    if (c.norm_out && blockIdx.x == 0 && threadIdx.x == 0) *c.norm_out = static_cast<float>(norm);
    const double coef = isinf(c.max_norm) ? 1.0 : c.max_norm / (norm + 1e-6);
    return coef >= 1.0 ? 1.f : static_cast<float>(coef);
}

template <int DT>
__device__ __forceinline__ void scale_block(void* p, const int64_t n, const int64_t e0, const float coef) {
    typedef typename Elem<DT>::type T;
    constexpr int VE = 16 / sizeof(T), TURNS = BLOCK_BYTES / (BLOCK * 16);
    T* g = static_cast<T*>(p);
    Vec<DT, VE> v[TURNS];
#pragma unroll
    for (int k = 0; k < TURNS; ++k) {
        const int64_t e = e0 + (k * BLOCK + threadIdx.x) * VE;
        if (e + VE <= n) v[k].load(g + e);
    }
#pragma unroll
    for (int k = 0; k < TURNS; ++k) {
        const int64_t e = e0 + (k * BLOCK + threadIdx.x) * VE;
        if (e + VE <= n) {
#pragma unroll
            for (int i = 0; i < VE; ++i) v[k].set(i, v[k].get(i) * coef);
            v[k].store(g + e);
        } else {
            for (int64_t i = e; i < n; ++i) g[i] = Elem<DT>::down(Elem<DT>::up(g[i]) * coef);
        }
    }
}

__global__ __launch_bounds__(BLOCK) void grad_scale_kernel(const GradArgs a, const int blocks, const Clip c) {
    __shared__ double lds[BLOCK / 64];
    const float coef = clip_coef(c, lds);
    for (int b = blockIdx.x; b < blocks; b += gridDim.x) {
        const int t = tensor_of(a, b);
        const int64_t k = b - a.first_block[t];
        if (a.dtype[t] == SPARC_F32) scale_block<SPARC_F32>(a.p[t], a.n[t], k * (BLOCK_BYTES / 4), coef);
        else if (a.dtype[t] == SPARC_BF16) scale_block<SPARC_BF16>(a.p[t], a.n[t], k * (BLOCK_BYTES / 2), coef);
        else scale_block<SPARC_F16>(a.p[t], a.n[t], k * (BLOCK_BYTES / 2), coef);
    }
}

struct AdamClipArgs {
    sparc_adam_tensor_t t[ADAM_MOST];
    int32_t first_block[ADAM_MOST + 1];
    int n_tensors;
    float step_size, bc2_rsqrt, beta2, one_minus_beta1, one_minus_beta2, eps, weight_decay;
};

// The update of sparc_adam_step for the gradient c g.
__device__ __forceinline__ void adam_one(float& p, const float g0, float& m, float& v, const AdamClipArgs& a, const float coef) {
    float g = coef * g0;
    if (a.weight_decay != 0.f) g = fmaf(a.weight_decay, p, g);
    m = fmaf(a.one_minus_beta1, g - m, m);
    v = fmaf(a.beta2, v, a.one_minus_beta2 * g * g);
    p -= a.step_size * (m / (sqrtf(v) * a.bc2_rsqrt + a.eps));
}

__global__ __launch_bounds__(BLOCK) void adam_clip_kernel(const AdamClipArgs a, const int blocks, const Clip c) {
    __shared__ double lds[BLOCK / 64];
    typedef Vec<SPARC_F32, 4> V4;
    const float coef = clip_coef(c, lds);
    for (int b = blockIdx.x; b < blocks; b += gridDim.x) {
        const int ti = tensor_of(a, b);
        const sparc_adam_tensor_t t = a.t[ti];
        const int64_t e = (static_cast<int64_t>(b) - a.first_block[ti]) * ADAM_ELEMS + threadIdx.x * 4;
        if (e + 4 <= t.n) {
            V4 p, g, m, v;
            p.load(t.p + e);
            g.load(t.g + e);
            m.load(t.m + e);
            v.load(t.v + e);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float pi = p.v[i], mi = m.v[i], vi = v.v[i];
                adam_one(pi, g.v[i], mi, vi, a, coef);
                p.v[i] = pi; m.v[i] = mi; v.v[i] = vi;
            }
            p.store(t.p + e);
            m.store(t.m + e);
            v.store(t.v + e);
        } else {
            for (int64_t i = e; i < t.n; ++i) {
                float p = t.p[i], m = t.m[i], v = t.v[i];
                adam_one(p, t.g[i], m, v, a, coef);
                t.p[i] = p; t.m[i] = m; t.v[i] = v;
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

// The first `count` tensors of t as kernel arguments; returns their number of blocks (below 2^30: SPARC_GRAD_MAX_ELEMS).
int64_t fill(GradArgs& a, const sparc_grad_tensor_t* t, const int count, const int block_bytes) {
    int64_t blocks = 0;
    for (int i = 0; i < count; ++i) {
        a.p[i] = t[i].p;
        a.n[i] = t[i].n;
        a.dtype[i] = static_cast<uint8_t>(t[i].dtype);
        a.first_block[i] = static_cast<int32_t>(blocks);
        const int64_t per = block_bytes / (t[i].dtype == SPARC_F32 ? 4 : 2);
        blocks += (t[i].n + per - 1) / per;
    }
    a.first_block[count] = static_cast<int32_t>(blocks);
    a.n_tensors = count;
    return blocks;
}

}  // namespace

extern "C" size_t sparc_grad_norm_workspace_bytes(int64_t n_tensors) {
    if (n_tensors < 0) return 0;
    const int64_t launches = (n_tensors + SPARC_GRAD_MAX_TENSORS - 1) / SPARC_GRAD_MAX_TENSORS;
    return static_cast<size_t>(launches > 0 ? launches : 1) * PARTS * sizeof(double);
}

extern "C" int sparc_grad_norm(int64_t n_tensors, const sparc_grad_tensor_t* tensors, double* parts, size_t parts_bytes,
                               int64_t* n_parts, sparc_stream_t stream) {
    if (!parts || !n_parts || !grads_ok(n_tensors, tensors)) return SPARC_ERR_ARG;
    if (parts_bytes < sparc_grad_norm_workspace_bytes(n_tensors) || (reinterpret_cast<uintptr_t>(parts) & 7)) return SPARC_ERR_WS;
    int64_t total = 0;
    int launches = 0;
    for (int64_t from = 0; from < n_tensors; from += SPARC_GRAD_MAX_TENSORS) {
        GradArgs a;
        const int count = static_cast<int>(n_tensors - from < SPARC_GRAD_MAX_TENSORS ? n_tensors - from : SPARC_GRAD_MAX_TENSORS);
        const int64_t blocks = fill(a, tensors + from, count, NORM_BYTES);
        if (blocks == 0) continue;
        const int grid = static_cast<int>(blocks < PARTS ? blocks : PARTS);
        hipLaunchKernelGGL(grad_squares_kernel, dim3(grid), dim3(NORM_THREADS), 0, stream, a, static_cast<int>(blocks), parts + total);
        SPARC_CHECK_LAUNCH();
        total += grid;
        ++launches;
    }
    if (launches > 1) {
        hipLaunchKernelGGL(grad_parts_kernel, dim3(1), dim3(BLOCK), 0, stream, parts, total);
        SPARC_CHECK_LAUNCH();
        total = 1;
    }
    *n_parts = total;
    return SPARC_OK;
}

extern "C" int sparc_grad_scale(int64_t n_tensors, const sparc_grad_tensor_t* tensors, const double* parts, int64_t n_parts,
                                double max_norm, float* norm_out, sparc_stream_t stream) {
    if (!parts || !norm_out || n_parts < 0 || n_parts > PARTS || !(max_norm >= 0.0) || !grads_ok(n_tensors, tensors)) return SPARC_ERR_ARG;
    Clip c = {parts, norm_out, max_norm, static_cast<int>(n_parts)};
    for (int64_t from = 0; from < n_tensors || from == 0; from += SPARC_GRAD_MAX_TENSORS) {
        GradArgs a;
        const int count = static_cast<int>(n_tensors - from < SPARC_GRAD_MAX_TENSORS ? n_tensors - from : SPARC_GRAD_MAX_TENSORS);
        const int64_t blocks = fill(a, tensors + from, count, BLOCK_BYTES);
        if (blocks == 0 && !c.norm_out) continue;
        const int grid = static_cast<int>(blocks < 1 ? 1 : blocks < MOST_BLOCKS ? blocks : MOST_BLOCKS);
        hipLaunchKernelGGL(grad_scale_kernel, dim3(grid), dim3(BLOCK), 0, stream, a, static_cast<int>(blocks), c);
        SPARC_CHECK_LAUNCH();
        c.norm_out = nullptr;
    }
    return SPARC_OK;
}

extern "C" int sparc_adam_step_clipped(int64_t n_tensors, const sparc_adam_tensor_t* tensors, double lr, double beta1, double beta2,
                                       double eps, double weight_decay, int64_t step, const double* parts, int64_t n_parts,
                                       double max_norm, float* norm_out, sparc_stream_t stream) {
    if (n_tensors < 0 || (n_tensors > 0 && !tensors) || step < 1 || !(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0) ||
        !(eps >= 0.0) || !parts || !norm_out || n_parts < 0 || n_parts > PARTS || !(max_norm >= 0.0))
        return SPARC_ERR_ARG;
    for (int64_t i = 0; i < n_tensors; ++i) {
        const sparc_adam_tensor_t& t = tensors[i];
        if (t.n < 0 || t.n > SPARC_GRAD_MAX_ELEMS || (t.n > 0 && (!t.p || !t.g || !t.m || !t.v))) return SPARC_ERR_ARG;
    }
    const double bc1 = 1.0 - pow(beta1, static_cast<double>(step)), bc2 = 1.0 - pow(beta2, static_cast<double>(step));
    Clip c = {parts, norm_out, max_norm, static_cast<int>(n_parts)};
    for (int64_t from = 0; from < n_tensors || from == 0; from += ADAM_MOST) {
        AdamClipArgs a;
        const int count = static_cast<int>(n_tensors - from < ADAM_MOST ? n_tensors - from : ADAM_MOST);
        int64_t blocks = 0;
        for (int i = 0; i < count; ++i) {
            a.t[i] = tensors[from + i];
            a.first_block[i] = static_cast<int32_t>(blocks);
            blocks += (a.t[i].n + ADAM_ELEMS - 1) / ADAM_ELEMS;
        }
        a.first_block[count] = static_cast<int32_t>(blocks);
        a.n_tensors = count;
        a.step_size = static_cast<float>(lr / bc1);
        a.bc2_rsqrt = static_cast<float>(1.0 / sqrt(bc2));
        a.beta2 = static_cast<float>(beta2);
        a.one_minus_beta1 = static_cast<float>(1.0 - beta1);
        a.one_minus_beta2 = static_cast<float>(1.0 - beta2);
        a.eps = static_cast<float>(eps);
        a.weight_decay = static_cast<float>(weight_decay);
        if (blocks == 0 && !c.norm_out) continue;
        const int grid = static_cast<int>(blocks < 1 ? 1 : blocks < MOST_BLOCKS ? blocks : MOST_BLOCKS);
        hipLaunchKernelGGL(adam_clip_kernel, dim3(grid), dim3(BLOCK), 0, stream, a, static_cast<int>(blocks), c);
        SPARC_CHECK_LAUNCH();
        c.norm_out = nullptr;
    }
    return SPARC_OK;
}
