// The global gradient norm over many tensors, clipping by it, and the Adam step that applies the
// clipping factor while it reads the gradients.
//
//   norm   N = sqrt(sum over tensors and elements of |g|^2)
//   clip   c = min(1, max_norm / (N + 1e-6)),  g <- c g
//   Adam   g' = c g (+ wd p),  m <- b1 m + (1 - b1) g',  v <- b2 v + (1 - b2) g'^2,
//          p <- (p - lr wd p) - lr / (1 - b1^t) * m / (sqrt(v / (1 - b2^t)) + eps)
//
// All three stream their tensors once through the SMs and are bound by HBM (small lists: by the
// launches).  The tensors' addresses travel as kernel parameters, so a call copies nothing to the
// device, keeps nothing, and can be captured: a table of up to kBigTable tensors goes into the
// 32 KB of parameters a launch may carry, and longer lists take several launches.
//
// Work is cut into units of kUnit (1024) elements, whatever their type, numbered through the whole
// list; a block takes one contiguous range of units, so neighbouring blocks do not depend on how
// the tensors' sizes fall, and walks it tensor by tensor.
//
// The norm is summed in two fixed stages (per-block partials, then every block that needs the
// norm adds the partials in the same order), so it is bitwise repeatable, with no atomics.  Sums
// are held in 64 bits: the squares of fp32 and bf16 gradients leave the fp32 range well before the
// gradients do.
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <vector>

#include "scx.h"
#include "scx_internal.h"
#include "scx_vec.cuh"

namespace {

using scx::from_f32;
using scx::to_f32;
using scx::Vec;

constexpr int kThreads = 256;
constexpr int kUnit = 1024;        // elements per unit
constexpr int kSmallTable = 32;    // tensors per launch, short lists
constexpr int kBigTable = 448;     // and long ones (24 KB of kernel parameters)
constexpr int kBlocksPerSm = 4;
constexpr int kDeep = 4;           // vectors of a thread in flight, clipping and long lists' norm
constexpr long long kManyUnits = 16384;
constexpr int kMaxSms = 256;       // sizes the workspace: one partial per block

enum : int { kF32 = 0, kBf16 = 1, kF16 = 2 };

template <int N>
struct ReadTable {
    const void* ptr[N];
    long long count[N];
    int first[N + 1];  // first unit of each tensor
    unsigned char dtype[N];
    int n;
};

template <int N>
struct StepTable {
    float* step[N];
};

template <int N>
struct AdamTable {
    void* p[N];
    const void* g[N];
    float* m[N];
    float* v[N];
    long long count[N];
    int first[N + 1];
    unsigned char dtype[N];
    int n;
    int base;  // index of the table's first tensor in the whole list
};

struct AdamScalars {
    float beta1, rest1, beta2, rest2;  // rest = 1 - beta, from the 64-bit beta (0.999 loses 1e-5 of it in fp32)
    float eps, weight_decay, shrink;   // shrink = lr * weight_decay where decoupled, else 0
    int decoupled;
};

__device__ __forceinline__ void grid_dep_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_dep_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// Sum over the block, the same bits in every thread.
__device__ double block_sum(double v) {
    __shared__ double part[kThreads / 32];
    __shared__ double total;
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = v;
    __syncthreads();
    if (threadIdx.x == 0) {
        double s = 0.0;
        for (int i = 0; i < kThreads / 32; ++i) s += part[i];
        total = s;
    }
    __syncthreads();
    return total;
}

// The tensor that unit u belongs to: the last one whose first unit is not after u, so never an
// empty one.
template <typename Table>
__device__ __forceinline__ int find_tensor(const Table& t, int u) {
    int lo = 0, hi = t.n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (t.first[mid] <= u) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Calls f(tensor, begin, end) for every piece of this block's range of units, from the last to the
// first where BACK: a pass behind the norm's takes first what that one read last, which is in L2
// (clipping 67M fp32 values: 173 us forwards, 139 us backwards and four vectors deep).
template <bool BACK = false, typename Table, typename F>
__device__ __forceinline__ void for_pieces(const Table& t, F f) {
    const long long units = t.first[t.n];
    int u = static_cast<int>(units * blockIdx.x / gridDim.x);
    int end = static_cast<int>(units * (blockIdx.x + 1) / gridDim.x);
    if (u >= end) return;
    if constexpr (BACK) {
        for (int k = find_tensor(t, end - 1); u < end; --k) {
            const int start = max(u, t.first[k]);
            const long long a = static_cast<long long>(start - t.first[k]) * kUnit;
            const long long b = min(t.count[k], static_cast<long long>(end - t.first[k]) * kUnit);
            f(k, a, b);
            end = start;
        }
    } else {
        for (int k = find_tensor(t, u); u < end; ++k) {
            const int stop = min(end, t.first[k + 1]);
            const long long a = static_cast<long long>(u - t.first[k]) * kUnit;
            const long long b = min(t.count[k], static_cast<long long>(stop - t.first[k]) * kUnit);
            f(k, a, b);
            u = stop;
        }
    }
}

// Elements before the first address of p that is a multiple of `bytes`.
template <typename T>
__device__ __forceinline__ int elements_to(const T* p, int bytes) {
    const unsigned r = static_cast<unsigned>(reinterpret_cast<uintptr_t>(p) % bytes);
    return r ? static_cast<int>((bytes - r) / sizeof(T)) : 0;
}

// AHEAD: the thread's next four vectors are under way while four are added, in the same order.  For fp32 alone:
// two-byte vectors have twice the sums to hide the reads behind (40M bf16 values: 18.9 us, 20.3 us ahead).
template <bool AHEAD, typename T>
__device__ double square_sum(const T* __restrict__ p, long long n) {
    constexpr int V = 16 / sizeof(T);
    double s = 0.0;
    const long long head = min(n, static_cast<long long>(elements_to(p, 16)));
    const long long body = (n - head) / V;
    const Vec<T, V>* q = reinterpret_cast<const Vec<T, V>*>(p + head);
    auto add = [&](const Vec<T, V> x) {
#pragma unroll
        for (int j = 0; j < V / 2; ++j) {
            const float2 two = x.pair(j);
            const double a = two.x, b = two.y;
            s = fma(a, a, s);
            s = fma(b, b, s);
        }
    };
    if constexpr (AHEAD && sizeof(T) == 4) {
        Vec<T, V> x[kDeep], y[kDeep];
        auto load = [&](Vec<T, V> (&to)[kDeep], long long i) {
#pragma unroll
            for (int d = 0; d < kDeep; ++d) {
                to[d] = Vec<T, V>{};
                if (i + d * kThreads < body) to[d] = q[i + d * kThreads];
            }
        };
        load(x, threadIdx.x);
        for (long long i = threadIdx.x; i < body; i += 2 * kDeep * kThreads) {
            load(y, i + kDeep * kThreads);
#pragma unroll
            for (int d = 0; d < kDeep; ++d) add(x[d]);
            load(x, i + 2 * kDeep * kThreads);
#pragma unroll
            for (int d = 0; d < kDeep; ++d) add(y[d]);
        }
    } else {
#pragma unroll 4
        for (long long i = threadIdx.x; i < body; i += kThreads) {
            const Vec<T, V> x = q[i];
            add(x);
        }
    }
    for (long long i = threadIdx.x; i < n - body * V; i += kThreads) {
        const double d = to_f32(p[i < head ? i : i + body * V]);
        s = fma(d, d, s);
    }
    return s;
}

// This thread's last index below n, its indices being threadIdx.x + k kThreads; negative without one.
__device__ __forceinline__ long long last_turn(long long n) {
    return threadIdx.x + (n - 1 - static_cast<long long>(threadIdx.x) + kThreads) / kThreads * kThreads - kThreads;
}

template <typename T>
__device__ void scale_piece(T* __restrict__ p, long long n, float c) {
    constexpr int V = 16 / sizeof(T);
    const long long head = min(n, static_cast<long long>(elements_to(p, 16)));
    const long long body = (n - head) / V;
    Vec<T, V>* q = reinterpret_cast<Vec<T, V>*>(p + head);
    for (long long i = last_turn(body); i >= 0; i -= kDeep * kThreads) {
        Vec<T, V> x[kDeep];
#pragma unroll
        for (int d = 0; d < kDeep; ++d)
            if (i >= d * kThreads) x[d] = q[i - d * kThreads];
#pragma unroll
        for (int d = 0; d < kDeep; ++d) {
            if (i < d * kThreads) break;
#pragma unroll
            for (int j = 0; j < V / 2; ++j) {
                const float2 two = x[d].pair(j);
                x[d].set_pair(j, make_float2(two.x * c, two.y * c));
            }
            q[i - d * kThreads] = x[d];
        }
    }
    for (long long i = threadIdx.x; i < n - body * V; i += kThreads) {
        T& e = p[i < head ? i : i + body * V];
        from_f32(e, to_f32(e) * c);
    }
}

// Per-block partial sums of squares.  In an Adam step block 0 also advances the tensors' step
// counts and leaves (lr / (1 - b1^t), 1 / sqrt(1 - b2^t)) of each in `corrections`.  AHEAD for lists of
// more than kManyUnits (67M fp32 values: 43 us, 47 us without; 2.4M: 7.4 us and 6.2 us without; the limit lies
// between the two lengths that were measured).
template <int N, bool STEPS, bool AHEAD>
__global__ void __launch_bounds__(kThreads) square_sum_kernel(const __grid_constant__ ReadTable<N> t,
                                                              const __grid_constant__ StepTable<STEPS ? N : 1> steps,
                                                              int nsteps, float2* corrections, double lr,
                                                              const float* lr_device, double beta1, double beta2,
                                                              double* partial) {
    grid_dep_launch();
    if (STEPS && blockIdx.x == 0) {
        const double rate = lr_device ? static_cast<double>(*lr_device) : lr;
        for (int i = threadIdx.x; i < nsteps; i += kThreads) {
            const float count = *steps.step[i] + 1.f;
            *steps.step[i] = count;
            const double k = count;
            corrections[i] = make_float2(static_cast<float>(rate / (1.0 - pow(beta1, k))),
                                         static_cast<float>(1.0 / sqrt(1.0 - pow(beta2, k))));
        }
    }
    if (partial == nullptr) return;
    double s = 0.0;
    for_pieces(t, [&](int k, long long a, long long b) {
        if (t.dtype[k] == kF32) s += square_sum<AHEAD>(static_cast<const float*>(t.ptr[k]) + a, b - a);
        else if (t.dtype[k] == kBf16) s += square_sum<AHEAD>(static_cast<const __nv_bfloat16*>(t.ptr[k]) + a, b - a);
        else s += square_sum<AHEAD>(static_cast<const __half*>(t.ptr[k]) + a, b - a);
    });
    s = block_sum(s);
    if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

// sqrt of the partials' sum; the same bits in every block and thread.
__device__ double total_norm(const double* partial, int parts) {
    double s = 0.0;
    for (int i = threadIdx.x; i < parts; i += kThreads) s += partial[i];
    return sqrt(block_sum(s));
}

// min(1, max_norm / (norm + 1e-6)); NaN stays NaN.
__device__ __forceinline__ float clip_factor(double norm, double max_norm) {
    const double c = max_norm / (norm + 1.0e-6);
    return c > 1.0 ? 1.f : static_cast<float>(c);
}

__global__ void __launch_bounds__(kThreads) norm_kernel(const double* partial, int parts, float* norm) {
    grid_dep_wait();
    const double total = total_norm(partial, parts);
    if (threadIdx.x == 0) *norm = static_cast<float>(total);
}

template <int N>
__global__ void __launch_bounds__(kThreads) clip_kernel(const __grid_constant__ ReadTable<N> t, const double* partial,
                                                        int parts, double max_norm, float* norm) {
    grid_dep_wait();
    const double total = total_norm(partial, parts);
    if (norm != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *norm = static_cast<float>(total);
    const float c = clip_factor(total, max_norm);
    if (c == 1.f) return;  // a product with one changes nothing
    for_pieces<true>(t, [&](int k, long long a, long long b) {
        void* p = const_cast<void*>(t.ptr[k]);
        if (t.dtype[k] == kF32) scale_piece(static_cast<float*>(p) + a, b - a, c);
        else if (t.dtype[k] == kBf16) scale_piece(static_cast<__nv_bfloat16*>(p) + a, b - a, c);
        else scale_piece(static_cast<__half*>(p) + a, b - a, c);
    });
}

__device__ __forceinline__ void adam_one(float& p, float g, float& m, float& v, float c, float2 k,
                                         const AdamScalars& s) {
    g *= c;
    if (!s.decoupled && s.weight_decay != 0.f) g = fmaf(s.weight_decay, p, g);  // no 0 * inf from an infinite p
    m = fmaf(s.beta1, m, s.rest1 * g);
    v = fmaf(s.beta2, v, s.rest2 * g * g);
    const float move = k.x * m / fmaf(sqrtf(v), k.y, s.eps);
    // the decay joins the update before p is rounded: lr * wd alone is often below half a step of p.  An infinite p
    // has no decay to take, and stays.
    p -= isinf(p) ? move : fmaf(s.shrink, p, move);
}

template <int DEEP, typename T>
__device__ void adam_piece(T* __restrict__ p, const T* __restrict__ g, float* __restrict__ m, float* __restrict__ v,
                           long long n, float c, float2 k, const AdamScalars& s) {
    constexpr int V = 4;
    const long long head = min(n, static_cast<long long>(elements_to(m, 16)));
    const bool even = reinterpret_cast<uintptr_t>(p + head) % (V * sizeof(T)) == 0 &&
                      reinterpret_cast<uintptr_t>(g + head) % (V * sizeof(T)) == 0 &&
                      reinterpret_cast<uintptr_t>(v + head) % 16 == 0;
    const long long body = even ? (n - head) / V : 0;
    auto* pv = reinterpret_cast<Vec<T, V>*>(p + head);
    auto* gv = reinterpret_cast<const Vec<T, V>*>(g + head);
    auto* mv = reinterpret_cast<Vec<float, V>*>(m + head);
    auto* vv = reinterpret_cast<Vec<float, V>*>(v + head);
    for (long long i = last_turn(body); i >= 0; i -= DEEP * kThreads) {
        Vec<T, V> pi[DEEP], gi[DEEP];
        Vec<float, V> mi[DEEP], vi[DEEP];
#pragma unroll
        for (int d = 0; d < DEEP; ++d) {
            if (i < d * kThreads) break;
            pi[d] = pv[i - d * kThreads];
            gi[d] = gv[i - d * kThreads];
            mi[d] = mv[i - d * kThreads];
            vi[d] = vv[i - d * kThreads];
        }
#pragma unroll
        for (int d = 0; d < DEEP; ++d) {
            if (i < d * kThreads) break;
#pragma unroll
            for (int j = 0; j < V / 2; ++j) {
                float2 two = pi[d].pair(j);
                const float2 g2 = gi[d].pair(j);
                adam_one(two.x, g2.x, mi[d].w[2 * j], vi[d].w[2 * j], c, k, s);
                adam_one(two.y, g2.y, mi[d].w[2 * j + 1], vi[d].w[2 * j + 1], c, k, s);
                pi[d].set_pair(j, two);
            }
            pv[i - d * kThreads] = pi[d];
            mv[i - d * kThreads] = mi[d];
            vv[i - d * kThreads] = vi[d];
        }
    }
    for (long long i = threadIdx.x; i < n - body * V; i += kThreads) {
        const long long e = i < head ? i : i + body * V;
        float x = to_f32(p[e]);
        adam_one(x, to_f32(g[e]), m[e], v[e], c, k, s);
        from_f32(p[e], x);
    }
}

// DEEP vectors of each tensor in flight per thread: two for long lists, whose stream they fill (67M values:
// 352 us, 373 us with one); one for short ones, where twice the blocks fit an SM (2.4M: 19 us, 21 us
// with two); the limit as above.
template <int N, int DEEP>
__global__ void __launch_bounds__(kThreads) adam_kernel(const __grid_constant__ AdamTable<N> t,
                                                        const float2* corrections, const double* partial, int parts,
                                                        const float* given_norm, double max_norm, float* norm,
                                                        AdamScalars s, double weight_decay,
                                                        const float* lr_device) {
    grid_dep_wait();
    float c = 1.f;
    if (given_norm != nullptr) {
        c = clip_factor(*given_norm, max_norm);
    } else if (partial != nullptr) {
        const double total = total_norm(partial, parts);
        if (norm != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *norm = static_cast<float>(total);
        c = clip_factor(total, max_norm);
    }
    if (lr_device && s.decoupled) s.shrink = static_cast<float>(static_cast<double>(*lr_device) * weight_decay);
    for_pieces<true>(t, [&](int i, long long a, long long b) {
        const float2 k = corrections[t.base + i];
        if (t.dtype[i] == kF32)
            adam_piece<DEEP>(static_cast<float*>(t.p[i]) + a, static_cast<const float*>(t.g[i]) + a, t.m[i] + a, t.v[i] + a,
                       b - a, c, k, s);
        else if (t.dtype[i] == kBf16)
            adam_piece<DEEP>(static_cast<__nv_bfloat16*>(t.p[i]) + a, static_cast<const __nv_bfloat16*>(t.g[i]) + a,
                       t.m[i] + a, t.v[i] + a, b - a, c, k, s);
        else
            adam_piece<DEEP>(static_cast<__half*>(t.p[i]) + a, static_cast<const __half*>(t.g[i]) + a, t.m[i] + a,
                       t.v[i] + a, b - a, c, k, s);
    });
}

// ---------------------------------------------------------------------------- host side

size_t element_size(int dtype) { return dtype == kF32 ? 4 : 2; }

struct Span {
    uintptr_t begin, end;
};

bool disjoint(std::vector<Span>& spans) {
    std::sort(spans.begin(), spans.end(), [](const Span& a, const Span& b) { return a.begin < b.begin; });
    for (size_t i = 1; i < spans.size(); ++i)
        if (spans[i].begin < spans[i - 1].end) return false;
    return true;
}

// Whether `one` shares memory with any of sorted, disjoint spans.
bool meets(const std::vector<Span>& spans, const Span& one) {
    const auto at = std::upper_bound(spans.begin(), spans.end(), one.begin,
                                     [](uintptr_t begin, const Span& s) { return begin < s.end; });
    return at != spans.end() && at->begin < one.end;
}

bool valid_tensor(const void* p, long long count, int dtype) {
    return count >= 0 && dtype >= kF32 && dtype <= kF16 && count <= (1LL << 40) &&
           (count == 0 || (p != nullptr && reinterpret_cast<uintptr_t>(p) % element_size(dtype) == 0));
}

Span span_of(const void* p, long long bytes) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(p);
    return {a, a + static_cast<uintptr_t>(bytes)};
}

int grid_for(long long units) {
    const int sms = std::min(scx::num_sms(), kMaxSms);
    return static_cast<int>(std::max(1LL, std::min(units, static_cast<long long>(sms) * kBlocksPerSm)));
}

constexpr int kMaxBlocks = kMaxSms * kBlocksPerSm;

int launches_for(size_t tensors) { return static_cast<int>((tensors + kBigTable - 1) / kBigTable); }

long long units_of(long long count) { return (count + kUnit - 1) / kUnit; }

template <int N>
bool fill(ReadTable<N>& t, int from, int n, const void* const* ptrs, const long long* counts, const int* dtypes) {
    t.n = std::min(n - from, N);
    long long units = 0;
    for (int k = 0; k < t.n; ++k) {
        const int i = from + k;
        t.ptr[k] = ptrs[i];
        t.count[k] = counts[i];
        t.dtype[k] = static_cast<unsigned char>(dtypes[i]);
        t.first[k] = static_cast<int>(units);
        units += units_of(counts[i]);
        if (units > (1LL << 30)) return false;
    }
    t.first[t.n] = static_cast<int>(units);
    return true;
}

struct StepArgs {
    float* const* steps = nullptr;
    float2* corrections = nullptr;
    double lr = 0.0, beta1 = 0.0, beta2 = 0.0;
    const float* lr_device = nullptr;
};

// Launches the partial sums of every table of the list; with steps, also their advance.  partial
// is null where no norm is wanted.  *parts: the number of partials written.
template <int N, bool STEPS>
cudaError_t launch_sums(int n, const void* const* ptrs, const long long* counts, const int* dtypes, const StepArgs& a,
                        double* partial, cudaStream_t s, int* parts) {
    *parts = 0;
    for (int from = 0; from < n; from += N) {
        ReadTable<N> t;
        StepTable<STEPS ? N : 1> st = {};
        if (!fill(t, from, n, ptrs, counts, dtypes)) return cudaErrorInvalidValue;
        if (STEPS)
            for (int k = 0; k < t.n; ++k) st.step[k] = a.steps[from + k];
        const int grid = partial ? grid_for(t.first[t.n]) : 1;
        const auto kernel = t.first[t.n] > kManyUnits ? square_sum_kernel<N, STEPS, true> : square_sum_kernel<N, STEPS, false>;
        kernel<<<grid, kThreads, 0, s>>>(t, st, t.n, a.corrections ? a.corrections + from : nullptr, a.lr, a.lr_device,
                                         a.beta1, a.beta2, partial ? partial + *parts : nullptr);
        const cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) return e;
        if (partial) *parts += grid;
    }
    return cudaSuccess;
}

// The launch after the sums: overlapped with their drain where one launch did all of them (a
// dependent launch waits for the one launch before it).
template <typename... P, typename... A>
cudaError_t launch_after(bool chained, void (*kernel)(P...), int grid, cudaStream_t s, A... args) {
    if (chained) return scx::launch_chained(kernel, dim3(grid), dim3(kThreads), 0, s, args...);
    kernel<<<grid, kThreads, 0, s>>>(args...);
    return cudaGetLastError();
}

template <int N>
cudaError_t launch_clip(int n, void* const* ptrs, const long long* counts, const int* dtypes, const double* partial,
                        int parts, double max_norm, float* norm, cudaStream_t s) {
    for (int from = 0; from < n; from += N) {
        ReadTable<N> t;
        if (!fill(t, from, n, ptrs, counts, dtypes)) return cudaErrorInvalidValue;
        const cudaError_t e = launch_after(n <= N, clip_kernel<N>, grid_for(t.first[t.n]), s, t, partial,
                                           parts, max_norm, from == 0 ? norm : nullptr);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

struct AdamLists {
    void* const* p;
    const void* const* g;
    float* const* m;
    float* const* v;
    const long long* counts;
    const int* dtypes;
};

template <int N>
cudaError_t launch_adam(int n, const AdamLists& l, const float2* corrections, const double* partial, int parts,
                        const float* given_norm, double max_norm, float* norm, const AdamScalars& sc, double weight_decay,
                        const float* lr_device, cudaStream_t s) {
    for (int from = 0; from < n; from += N) {
        AdamTable<N> t;
        t.n = std::min(n - from, N);
        t.base = from;
        long long units = 0;
        for (int k = 0; k < t.n; ++k) {
            const int i = from + k;
            t.p[k] = l.p[i];
            t.g[k] = l.g[i];
            t.m[k] = l.m[i];
            t.v[k] = l.v[i];
            t.count[k] = l.counts[i];
            t.dtype[k] = static_cast<unsigned char>(l.dtypes[i]);
            t.first[k] = static_cast<int>(units);
            units += units_of(l.counts[i]);
            if (units > (1LL << 30)) return cudaErrorInvalidValue;
        }
        t.first[t.n] = static_cast<int>(units);
        const cudaError_t e = launch_after(n <= N, units > kManyUnits ? adam_kernel<N, 2> : adam_kernel<N, 1>, grid_for(units), s, t, corrections, partial, parts,
                                           given_norm, max_norm, from == 0 ? norm : nullptr, sc, weight_decay, lr_device);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

size_t partial_bytes(size_t tensors) {
    return static_cast<size_t>(std::max(1, launches_for(tensors))) * kMaxBlocks * sizeof(double);
}

cudaError_t norm_or_clip(int n, void* const* ptrs, const long long* counts, const int* dtypes, bool clip,
                         double max_norm, float* norm, void* workspace, size_t bytes, cudaStream_t s) {
    if (n < 0 || (n > 0 && (!ptrs || !counts || !dtypes)) || norm == nullptr || workspace == nullptr ||
        reinterpret_cast<uintptr_t>(workspace) % 16 != 0 || reinterpret_cast<uintptr_t>(norm) % 4 != 0 ||
        bytes < partial_bytes(static_cast<size_t>(n)) || (clip && !(max_norm >= 0.0)))
        return cudaErrorInvalidValue;
    for (int i = 0; i < n; ++i)
        if (!valid_tensor(ptrs[i], counts[i], dtypes[i])) return cudaErrorInvalidValue;
    if (clip) {
        std::vector<Span> spans;
        for (int i = 0; i < n; ++i)
            if (counts[i] > 0)
                spans.push_back(span_of(ptrs[i], counts[i] * static_cast<long long>(element_size(dtypes[i]))));
        if (!disjoint(spans)) return cudaErrorInvalidValue;
    }
    double* partial = static_cast<double*>(workspace);
    int parts = 0;
    const bool small = n <= kSmallTable;
    const cudaError_t e = small ? launch_sums<kSmallTable, false>(n, ptrs, counts, dtypes, StepArgs{}, partial, s, &parts)
                                : launch_sums<kBigTable, false>(n, ptrs, counts, dtypes, StepArgs{}, partial, s, &parts);
    if (e != cudaSuccess) return e;
    if (!clip || n == 0) return launch_after(n > 0 && n <= kBigTable, norm_kernel, 1, s, partial, parts, norm);
    return small ? launch_clip<kSmallTable>(n, ptrs, counts, dtypes, partial, parts, max_norm, norm, s)
                 : launch_clip<kBigTable>(n, ptrs, counts, dtypes, partial, parts, max_norm, norm, s);
}

size_t align256(size_t b) { return (b + 255) / 256 * 256; }

cudaError_t adam(int n, const AdamLists& l, float* const* steps, double lr, const float* lr_device, double beta1,
                 double beta2, double eps, double weight_decay, int decoupled, double max_norm, const float* given_norm,
                 float* norm, void* workspace, size_t bytes, cudaStream_t s) {
    const bool clip = norm != nullptr;  // by the norm of these gradients
    if (n < 0 || (n > 0 && (!l.p || !l.g || !l.m || !l.v || !steps || !l.counts || !l.dtypes)) ||
        workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 16 != 0 ||
        bytes < scx_adam_workspace_size(n) || !std::isfinite(lr) || !(beta1 >= 0.0 && beta1 < 1.0) ||
        !(beta2 >= 0.0 && beta2 < 1.0) || !(eps >= 0.0) || !std::isfinite(weight_decay) ||
        (clip && given_norm != nullptr) ||
        ((clip || given_norm != nullptr) && !(max_norm >= 0.0)) || reinterpret_cast<uintptr_t>(norm) % 4 != 0)
        return cudaErrorInvalidValue;
    std::vector<Span> spans;
    for (int i = 0; i < n; ++i) {
        const long long c = l.counts[i];
        if (!valid_tensor(l.p[i], c, l.dtypes[i]) || !valid_tensor(l.g[i], c, l.dtypes[i]) ||
            !valid_tensor(l.m[i], c, kF32) || !valid_tensor(l.v[i], c, kF32) || !steps[i] ||
            reinterpret_cast<uintptr_t>(steps[i]) % 4 != 0)
            return cudaErrorInvalidValue;
        spans.push_back(span_of(steps[i], 4));
        if (c == 0) continue;
        spans.push_back(span_of(l.p[i], c * static_cast<long long>(element_size(l.dtypes[i]))));
        spans.push_back(span_of(l.m[i], c * 4));
        spans.push_back(span_of(l.v[i], c * 4));
    }
    if (!disjoint(spans)) return cudaErrorInvalidValue;
    for (int i = 0; i < n; ++i)  // a gradient is read while other blocks write
        if (l.counts[i] > 0 && meets(spans, span_of(l.g[i], l.counts[i] * static_cast<long long>(element_size(l.dtypes[i])))))
            return cudaErrorInvalidValue;
    const AdamScalars sc = {static_cast<float>(beta1), static_cast<float>(1.0 - beta1), static_cast<float>(beta2),
                            static_cast<float>(1.0 - beta2), static_cast<float>(eps), static_cast<float>(weight_decay),
                            decoupled ? static_cast<float>(lr * weight_decay) : 0.f, decoupled ? 1 : 0};
    float2* corrections = static_cast<float2*>(workspace);
    double* partial = clip ? reinterpret_cast<double*>(static_cast<char*>(workspace) +
                                                       align256(static_cast<size_t>(n) * sizeof(float2)))
                           : nullptr;
    const StepArgs a = {steps, corrections, lr, beta1, beta2, lr_device};
    int parts = 0;
    if (n == 0) return clip ? launch_after(false, norm_kernel, 1, s, partial, 0, norm) : cudaSuccess;
    const bool small = n <= kSmallTable;
    const cudaError_t e = small ? launch_sums<kSmallTable, true>(n, l.g, l.counts, l.dtypes, a, partial, s, &parts)
                                : launch_sums<kBigTable, true>(n, l.g, l.counts, l.dtypes, a, partial, s, &parts);
    if (e != cudaSuccess) return e;
    return small ? launch_adam<kSmallTable>(n, l, corrections, partial, parts, given_norm, max_norm, norm, sc,
                                            weight_decay, lr_device, s)
                 : launch_adam<kBigTable>(n, l, corrections, partial, parts, given_norm, max_norm, norm, sc,
                                          weight_decay, lr_device, s);
}

}  // namespace

extern "C" size_t scx_grad_norm_workspace_size(int n_tensors) {
    return n_tensors < 0 ? 0 : partial_bytes(static_cast<size_t>(n_tensors));
}

extern "C" int scx_grad_norm(int n_tensors, const void* const* tensors, const long long* counts, const int* dtypes,
                             float* norm, void* workspace, size_t workspace_bytes, scx_stream_t stream) {
    try {
        return norm_or_clip(n_tensors, const_cast<void* const*>(tensors), counts,
                            dtypes, false, 0.0, norm, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
    } catch (...) {
        return cudaErrorMemoryAllocation;
    }
}

extern "C" int scx_grad_clip(int n_tensors, void* const* tensors, const long long* counts, const int* dtypes,
                             double max_norm, float* norm, void* workspace, size_t workspace_bytes,
                             scx_stream_t stream) {
    try {
        return norm_or_clip(n_tensors, tensors, counts, dtypes, true, max_norm, norm, workspace, workspace_bytes,
                            static_cast<cudaStream_t>(stream));
    } catch (...) {
        return cudaErrorMemoryAllocation;
    }
}

extern "C" size_t scx_adam_workspace_size(int n_tensors) {
    if (n_tensors < 0) return 0;
    const size_t n = static_cast<size_t>(n_tensors);
    return align256(n * sizeof(float2)) + partial_bytes(n);
}

extern "C" int scx_adam_step(int n_tensors, void* const* params, const void* const* grads, float* const* exp_avgs,
                             float* const* exp_avg_sqs, float* const* steps, const long long* counts,
                             const int* dtypes, double lr, const float* lr_device, double beta1, double beta2,
                             double eps, double weight_decay, int decoupled, double max_norm,
                             const float* given_norm, float* norm, void* workspace, size_t workspace_bytes, scx_stream_t stream) {
    try {
        return adam(n_tensors, AdamLists{params, grads, exp_avgs, exp_avg_sqs, counts, dtypes}, steps, lr, lr_device,
                    beta1, beta2, eps, weight_decay, decoupled, max_norm, given_norm, norm, workspace, workspace_bytes,
                    static_cast<cudaStream_t>(stream));
    } catch (...) {
        return cudaErrorMemoryAllocation;
    }
}
