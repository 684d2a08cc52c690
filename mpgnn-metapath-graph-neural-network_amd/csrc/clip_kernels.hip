// The global norm over a list of gradient tensors and the gradients scaled to at most max_norm:
//   norm = (sum over every tensor of g^2)^(1/2)  or  max |g|
//   out  = g * min(1, max_norm / (norm + 1e-6))
// Bound by memory: each gradient is read for the norm, read again and written for the scaling
// (the second read comes from the 256 MB last-level cache while the list fits it).
//
// Each square is taken and summed in double, where no fp32 value's overflows or vanishes: the norm is the exact one
// rounded once to fp32. (Summing a vector's four or eight squares in fp32 first saves conversions and no time: 31 MB
// in 8.5 us so, 8.0 without.) Each thread adds its elements in order, then lanes, waves, workgroups, always in the
// same order: the norm does not change from run to run.
//
// Two kernels per list of up to kClipMax tensors (the tensor table is the kernel's argument, so a captured
// graph holds it by value): the norm kernel leaves one partial sum per workgroup, the scaling
// kernel's workgroups each add all partials (up to 2,048 doubles from L2) and so need no counter, no
// atomic and no third launch. With more than one list, one more workgroup adds the partials of all
// before the scaling. Tensors of at most kClipSmallBytes together take one launch of one workgroup.
//
// Measured, norm and scaling, averages: 31 MB of gradients 8.0 + 17.5 us; 400 tensors of 537 MB, four lists, 4 x (41 +
// 56) us (a read of all of them and a copy at 4.96 TB/s: 324 us).
#include <algorithm>
#include <vector>

#include "num_types.h"

namespace mpgnn {
namespace {

constexpr int kClipThreads = 256;
constexpr int kClipMax = 120;              // tensors per launch: 3.6 KB of kernel arguments
constexpr int kClipUnit = 16384;           // bytes of a tensor that a workgroup takes at a time
constexpr int kClipMaxLists = 1024;
constexpr int kClipBlocks = 2048;          // workgroups of a launch: eight per CU, all there at once
constexpr int kClipSmallThreads = 1024;
constexpr int64_t kClipSmallBytes = 32 * 1024;

struct ClipList {
    int n;
    int reversed;                    // units walked from the last one down
    int32_t unit_off[kClipMax + 1];  // tensor t owns units [unit_off[t], unit_off[t + 1])
    const void* g[kClipMax];
    void* o[kClipMax];
    int64_t numel[kClipMax];
    uint8_t dtype[kClipMax];
};

struct SumSq {
    typedef double acc;
    static __device__ __forceinline__ acc add(acc a, float v) { return __builtin_fma((double)v, (double)v, a); }
    template <int V>
    static __device__ __forceinline__ acc add_vec(acc a, const float (&v)[V]) {
        acc s = (double)v[0] * (double)v[0];
#pragma unroll
        for (int j = 1; j < V; ++j) s = add(s, v[j]);
        return a + s;
    }
    static __device__ __forceinline__ acc join(acc a, acc b) { return a + b; }
    static __device__ __forceinline__ double norm(acc a) { return ::sqrt(a); }
};

struct MaxAbs {  // a NaN anywhere stays
    typedef double acc;
    static __device__ __forceinline__ acc join(acc a, acc b) { return (b > a || b != b) ? b : a; }
    static __device__ __forceinline__ acc add(acc a, float v) { return join(a, (double)__builtin_fabsf(v)); }
    template <int V>
    static __device__ __forceinline__ acc add_vec(acc a, const float (&v)[V]) {
        float m = __builtin_fabsf(v[0]);
#pragma unroll
        for (int j = 1; j < V; ++j) {
            const float b = __builtin_fabsf(v[j]);
            m = (b > m || b != b) ? b : m;
        }
        return join(a, (double)m);
    }
    static __device__ __forceinline__ double norm(acc a) { return a; }
};

// A unit of a tensor: its whole vectors of 16 bytes (those of a thread asked for together), then the last
// elements of the tensor; tensors that are not aligned to 16 bytes go element by element.
template <typename T, int THREADS>
struct Unit {
    static constexpr int V = 16 / sizeof(T), U = kClipUnit / sizeof(T), N = U / (THREADS * V);
    int64_t e0, end;

    __device__ __forceinline__ Unit(int64_t numel, int64_t unit) : e0(unit * U), end(min(e0 + U, numel)) {}
    __device__ __forceinline__ int64_t at(int i) const { return e0 + (i * THREADS + (int)threadIdx.x) * V; }
    __device__ __forceinline__ bool whole(int i) const { return at(i) + V <= end; }
    __device__ __forceinline__ void load(float (&v)[N][V], const T* g) const {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (whole(i)) load_vec<T, V>(v[i], g + at(i));
    }
    __device__ __forceinline__ int64_t tail() const {  // this thread's element behind the whole vectors, or end
        const int64_t e = end - (end - e0) % V + (int)threadIdx.x;
        return e < end ? e : end;
    }
};

template <typename T, typename OP, int THREADS>
__device__ __forceinline__ typename OP::acc unit_norm(const T* g, int64_t numel, int64_t unit, typename OP::acc a) {
    typedef Unit<T, THREADS> X;
    const X u(numel, unit);
    if ((reinterpret_cast<uintptr_t>(g) & 15) == 0) {
        float v[X::N][X::V];
        u.load(v, g);
#pragma unroll
        for (int i = 0; i < X::N; ++i)
            if (u.whole(i)) a = OP::template add_vec<X::V>(a, v[i]);
        if (u.tail() < u.end) a = OP::add(a, (float)g[u.tail()]);
    } else {
#pragma unroll 8
        for (int64_t e = u.e0 + threadIdx.x; e < u.end; e += THREADS) a = OP::add(a, (float)g[e]);
    }
    return a;
}

template <typename T, int THREADS>
__device__ __forceinline__ void unit_scale(const T* g, T* o, int64_t numel, int64_t unit, float c) {
    typedef Unit<T, THREADS> X;
    const X u(numel, unit);
    if (((reinterpret_cast<uintptr_t>(g) | reinterpret_cast<uintptr_t>(o)) & 15) == 0) {
        float v[X::N][X::V];
        u.load(v, g);
#pragma unroll
        for (int i = 0; i < X::N; ++i) {
            if (!u.whole(i)) continue;
#pragma unroll
            for (int j = 0; j < X::V; ++j) v[i][j] *= c;
            store_vec<T, X::V>(o + u.at(i), v[i]);
        }
        const int64_t e = u.tail();
        if (e < u.end) o[e] = (T)((float)g[e] * c);
    } else {
#pragma unroll 8
        for (int64_t e = u.e0 + threadIdx.x; e < u.end; e += THREADS) o[e] = (T)((float)g[e] * c);
    }
}

template <typename OP, int THREADS>
__device__ __forceinline__ typename OP::acc block_join(typename OP::acc a, double* lds) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) a = OP::join(a, __shfl_xor(a, d, 64));
    const int wave = threadIdx.x / 64;
    if (threadIdx.x % 64 == 0) lds[wave] = a;
    __syncthreads();
    a = lds[0];
    for (int w = 1; w < THREADS / 64; ++w) a = OP::join(a, lds[w]);
    __syncthreads();
    return a;
}

// min(1, max_norm / (norm + 1e-6)) with a NaN kept, as a comparison with it is false
__device__ __forceinline__ float clip_factor(double norm, float max_norm) {
    const float c = max_norm / ((float)norm + 1e-6f);
    return c > 1.0f ? 1.0f : c;
}

// Units [beg, end) of the list, each with its tensor: f(tensor, unit within it).
template <typename F>
__device__ __forceinline__ void walk_units(const ClipList& L, const int32_t* s_off, int beg, int end, F&& f) {
    if (beg >= end) return;
    int lo = 0, hi = L.n;  // the tensor of unit beg: s_off[lo] <= beg < s_off[lo + 1]
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (s_off[mid] <= beg) lo = mid; else hi = mid;
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    for (int u = beg; u < end; ++u) {
        while (u >= L.unit_off[lo + 1]) ++lo;
        f(lo, (int64_t)(u - L.unit_off[lo]));
    }
}

template <typename OP, int THREADS>
__device__ __forceinline__ typename OP::acc range_norm(const ClipList& L, const int32_t* s_off, int beg, int end) {
    typename OP::acc a = 0;
    walk_units(L, s_off, beg, end, [&](int t, int64_t unit) {
        if (L.dtype[t] == MPGNN_F32)
            a = unit_norm<float, OP, THREADS>((const float*)L.g[t], L.numel[t], unit, a);
        else if (L.dtype[t] == MPGNN_BF16)
            a = unit_norm<__bf16, OP, THREADS>((const __bf16*)L.g[t], L.numel[t], unit, a);
        else
            a = unit_norm<_Float16, OP, THREADS>((const _Float16*)L.g[t], L.numel[t], unit, a);
    });
    return a;
}

template <int THREADS>
__device__ __forceinline__ void range_scale(const ClipList& L, const int32_t* s_off, int beg, int end, float c) {
    walk_units(L, s_off, beg, end, [&](int t, int64_t unit) {
        if (c == 1.0f && L.o[t] == L.g[t]) return;  // in place and not clipped: every product is the element
        if (L.dtype[t] == MPGNN_F32)
            unit_scale<float, THREADS>((const float*)L.g[t], (float*)L.o[t], L.numel[t], unit, c);
        else if (L.dtype[t] == MPGNN_BF16)
            unit_scale<__bf16, THREADS>((const __bf16*)L.g[t], (__bf16*)L.o[t], L.numel[t], unit, c);
        else
            unit_scale<_Float16, THREADS>((const _Float16*)L.g[t], (_Float16*)L.o[t], L.numel[t], unit, c);
    });
}

template <typename OP>
__global__ __launch_bounds__(kClipThreads) void clip_norm_kernel(ClipList L, int per_block, double* partials) {
    __shared__ int32_t s_off[kClipMax + 1];
    __shared__ double s_red[kClipThreads / 64];
    for (int i = threadIdx.x; i <= L.n; i += kClipThreads) s_off[i] = L.unit_off[i];
    __syncthreads();
    const int beg = blockIdx.x * per_block, end = min(beg + per_block, s_off[L.n]);
    const double a = block_join<OP, kClipThreads>(range_norm<OP, kClipThreads>(L, s_off, beg, end), s_red);
    if (threadIdx.x == 0) partials[blockIdx.x] = a;
}

template <typename OP>
__device__ __forceinline__ double join_partials(const double* partials, int n, double* s_red) {
    double a = 0;
    for (int i = threadIdx.x; i < n; i += kClipThreads) a = OP::join(a, partials[i]);
    return OP::norm(block_join<OP, kClipThreads>(a, s_red));
}

// the partials of several lists into the first (each thread reads its own before any is overwritten)
template <typename OP>
__global__ __launch_bounds__(kClipSmallThreads) void clip_join_kernel(double* partials, int n) {
    __shared__ double s_red[kClipSmallThreads / 64];
    double a = 0;
#pragma unroll 4
    for (int i = threadIdx.x; i < n; i += kClipSmallThreads) a = OP::join(a, partials[i]);
    a = block_join<OP, kClipSmallThreads>(a, s_red);
    if (threadIdx.x == 0) partials[0] = a;
}

// scale = 0: the norm alone
template <typename OP>
__global__ __launch_bounds__(kClipThreads) void clip_scale_kernel(ClipList L, int per_block, const double* partials,
                                                                   int n_partials, float max_norm, float* norm_out,
                                                                   int scale) {
    __shared__ int32_t s_off[kClipMax + 1];
    __shared__ double s_red[kClipThreads / 64];
    for (int i = threadIdx.x; i <= L.n; i += kClipThreads) s_off[i] = L.unit_off[i];
    const double norm = join_partials<OP>(partials, n_partials, s_red);
    if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
    if (!scale) return;
    const int b = L.reversed ? (int)gridDim.x - 1 - (int)blockIdx.x : (int)blockIdx.x;
    const int beg = b * per_block, end = min(beg + per_block, s_off[L.n]);
    range_scale<kClipThreads>(L, s_off, beg, end, clip_factor(norm, max_norm));
}

template <typename OP>
__global__ __launch_bounds__(kClipSmallThreads) void clip_small_kernel(ClipList L, float max_norm, float* norm_out,
                                                                        int scale) {
    __shared__ int32_t s_off[kClipMax + 1];
    __shared__ double s_red[kClipSmallThreads / 64];
    for (int i = threadIdx.x; i <= L.n; i += kClipSmallThreads) s_off[i] = L.unit_off[i];
    __syncthreads();
    const double norm = OP::norm(block_join<OP, kClipSmallThreads>(
        range_norm<OP, kClipSmallThreads>(L, s_off, 0, s_off[L.n]), s_red));
    if (threadIdx.x == 0) *norm_out = (float)norm;
    if (scale) range_scale<kClipSmallThreads>(L, s_off, 0, s_off[L.n], clip_factor(norm, max_norm));
}

int64_t tensor_units(const mpgnn_clip_tensor& t) {
    return (t.numel * dtype_bytes(t.dtype) + kClipUnit - 1) / kClipUnit;
}

// Does one of the tensors that a launch writes share memory with another that it writes, or with one that it reads
// other than as a whole in place? Workgroups would then read what others have scaled already.
bool shared_memory(const mpgnn_clip_tensor* tensors, int32_t n) {
    struct Range {
        uintptr_t lo, hi;
    };
    std::vector<Range> out;
    out.reserve(n);
    auto range = [](const mpgnn_clip_tensor& t, const void* p) {
        const uintptr_t lo = reinterpret_cast<uintptr_t>(p);
        return Range{lo, lo + (uintptr_t)(t.numel * dtype_bytes(t.dtype))};
    };
    for (int32_t k = 0; k < n; ++k)
        if (tensors[k].numel > 0) out.push_back(range(tensors[k], tensors[k].out));
    const auto before = [](const Range& a, const Range& b) { return a.lo < b.lo; };
    if (!std::is_sorted(out.begin(), out.end(), before)) std::sort(out.begin(), out.end(), before);
    for (size_t i = 1; i < out.size(); ++i)
        if (out[i].lo < out[i - 1].hi) return true;
    for (int32_t k = 0; k < n; ++k) {
        const mpgnn_clip_tensor& t = tensors[k];
        if (t.numel == 0 || t.grad == t.out) continue;  // in place: compared with the others above
        const Range g = range(t, t.grad);
        // the outputs are apart, so their ends are in order too: the first that ends behind the beginning
        const auto at = std::upper_bound(out.begin(), out.end(), g.lo, [](uintptr_t v, const Range& r) { return v < r.hi; });
        if (at != out.end() && at->lo < g.hi) return true;
    }
    return false;
}

template <typename OP>
int32_t clip_run(const mpgnn_clip_tensor* tensors, int32_t n, float max_norm, int32_t scale, float* norm, void* ws,
                 hipStream_t strm) {
    int64_t bytes = 0;
    int filled = 0;
    for (int k = 0; k < n; ++k) {
        filled += tensors[k].numel > 0;
        bytes += tensors[k].numel * dtype_bytes(tensors[k].dtype);
    }
    // the next up to kClipMax tensors with elements, from tensor `at` on; returns their units
    auto fill = [&](ClipList& L, int& at) {
        int32_t u = 0;
        L.n = 0;
        for (; at < n && L.n < kClipMax; ++at) {
            const mpgnn_clip_tensor& t = tensors[at];
            if (t.numel == 0) continue;
            L.unit_off[L.n] = u;
            L.g[L.n] = t.grad;
            L.o[L.n] = t.out;
            L.numel[L.n] = t.numel;
            L.dtype[L.n] = (uint8_t)t.dtype;
            u += (int32_t)tensor_units(t);
            ++L.n;
        }
        L.unit_off[L.n] = u;
        return (int64_t)u;
    };
    ClipList L{};
    if (filled <= kClipMax && bytes <= kClipSmallBytes) {
        int at = 0;
        fill(L, at);
        hipLaunchKernelGGL(clip_small_kernel<OP>, dim3(1), dim3(kClipSmallThreads), 0, strm, L, max_norm, norm, scale);
        return launch_status("clip: the launch failed");
    }
    const int lists = (filled + kClipMax - 1) / kClipMax;
    // units a workgroup
    auto share = [](int64_t u) { return (int)((u + kClipBlocks - 1) / kClipBlocks); };
    double* partials = static_cast<double*>(ws);
    int start[kClipMaxLists];  // the first tensor of each list
    int np = 0, at = 0;
    for (int l = 0; l < lists; ++l) {
        start[l] = at;
        const int64_t u = fill(L, at);
        const int per_block = share(u), blocks = (int)((u + per_block - 1) / per_block);
        hipLaunchKernelGGL(clip_norm_kernel<OP>, dim3(blocks), dim3(kClipThreads), 0, strm, L, per_block, partials + np);
        np += blocks;
    }
    if (lists > 1) {
        hipLaunchKernelGGL(clip_join_kernel<OP>, dim3(1), dim3(kClipSmallThreads), 0, strm, partials, np);
        np = 1;
    }
    // the lists from the last one down, each from its last unit down: what was read last is still
    // in the last-level cache
    for (int l = lists - 1; l >= 0; --l) {
        at = start[l];
        const int64_t u = fill(L, at);
        L.reversed = 1;
        const int per_block = share(u), blocks = scale ? (int)((u + per_block - 1) / per_block) : 1;
        hipLaunchKernelGGL(clip_scale_kernel<OP>, dim3(blocks), dim3(kClipThreads), 0, strm, L, per_block, partials, np,
                           max_norm, l == lists - 1 ? norm : nullptr, scale);
        if (!scale) break;
    }
    return launch_status("clip: a launch failed");
}

}  // namespace
}  // namespace mpgnn

extern "C" int32_t mpgnn_clip_workspace_bytes(int32_t n, int64_t* bytes) {
    using namespace mpgnn;
    if (n < 0 || !bytes) return arg_error("mpgnn_clip_workspace_bytes: negative n or bytes is null");
    if (n > kClipMax * kClipMaxLists) return unsupported("mpgnn_clip_workspace_bytes: more than 122,880 tensors");
    *bytes = (int64_t)std::max(1, (n + kClipMax - 1) / kClipMax) * kClipBlocks * (int64_t)sizeof(double);
    return MPGNN_OK;
}

extern "C" int32_t mpgnn_clip_by_global_norm(const mpgnn_clip_tensor* tensors, int32_t n, int32_t norm_kind,
                                             double max_norm, float* norm, void* workspace, void* stream) {
    using namespace mpgnn;
    if (n <= 0 || !tensors) return arg_error("mpgnn_clip_by_global_norm: no tensors");
    if (!norm || !workspace) return arg_error("mpgnn_clip_by_global_norm: norm or workspace is null");
    if (norm_kind != MPGNN_NORM_2 && norm_kind != MPGNN_NORM_INF)
        return arg_error("mpgnn_clip_by_global_norm: norm_kind is neither MPGNN_NORM_2 nor MPGNN_NORM_INF");
    if (n > kClipMax * kClipMaxLists) return unsupported("mpgnn_clip_by_global_norm: more than 122,880 tensors");
    int64_t units = 0;
    int32_t with_out = 0;
    for (int k = 0; k < n; ++k) {
        const mpgnn_clip_tensor& t = tensors[k];
        const int eb = dtype_bytes(t.dtype);
        if (!eb) return arg_error("mpgnn_clip_by_global_norm: unknown dtype");
        if (t.numel < 0 || (t.numel > 0 && !t.grad)) return arg_error("mpgnn_clip_by_global_norm: bad tensor");
        if (reinterpret_cast<uintptr_t>(t.grad) % eb || reinterpret_cast<uintptr_t>(t.out) % eb)
            return arg_error("mpgnn_clip_by_global_norm: a pointer is not aligned to its elements");
        if (t.numel > (int64_t{1} << 40)) return unsupported("mpgnn_clip_by_global_norm: over 2^40 elements");
        if (t.numel > 0 && t.out) ++with_out;
        else if (t.numel > 0 && with_out) return arg_error("mpgnn_clip_by_global_norm: out given for some tensors only");
        units += tensor_units(t);
    }
    int32_t nonempty = 0;
    for (int k = 0; k < n; ++k) nonempty += tensors[k].numel > 0;
    if (with_out && with_out != nonempty)
        return arg_error("mpgnn_clip_by_global_norm: out given for some tensors only");
    if (units > INT32_MAX) return unsupported("mpgnn_clip_by_global_norm: over 2^31 units of 16 KB");
    if (with_out) {
        try {
            if (shared_memory(tensors, n))
                return arg_error("mpgnn_clip_by_global_norm: an out overlaps another tensor of the list (scaled twice, or "
                                 "read after it was scaled)");
        } catch (...) {
            set_last_error_cstr("mpgnn_clip_by_global_norm: out of host memory");
            return MPGNN_ERR_ALLOC;
        }
    }
    hipStream_t strm = static_cast<hipStream_t>(stream);
    const float mn = (float)max_norm;
    return norm_kind == MPGNN_NORM_2 ? clip_run<SumSq>(tensors, n, mn, with_out > 0, norm, workspace, strm)
                                     : clip_run<MaxAbs>(tensors, n, mn, with_out > 0, norm, workspace, strm);
}
