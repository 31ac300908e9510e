// The residual-norm kernels for fields, [batch][channels][length]: a position's channels lie
// `length` elements apart, so a warp takes neighbouring positions of a few channels, and a block's
// warps together all channels of a tile of positions.
//
// A thread has V neighbouring positions (one vector load) of EPT channels, and keeps them in
// registers from the first load to the last store: every tensor is read once.  A warp's 32 lanes
// are 32/LC groups of positions x LC groups of channels; LC > 1 serves channel counts that would
// take more than 16 warps.  A statistic is a sum over a position's channel groups: each group
// leaves its part in shared memory, one thread per position adds them and leaves the result.
// The layer kind's variance is not taken from sums of squares: a group leaves its mean and its sum of
// squares about it, and the parts are joined about the common mean.
#include <algorithm>

#include "scx_internal.h"
#include "scx_residual_norm.cuh"

namespace scx_rn {
namespace {

constexpr int kMaxWarps = 16;
enum : int { kPostW = 0, kPostB = 1, kPreW = 2, kPreB = 3, kScaleW = 4, kVectors = 5 };

template <int V, int EPT, int LC>
struct Shape {
    static constexpr int kGroups = kMaxWarps * LC;  // most channel groups of a block
    static constexpr int kPos = 32 / LC * V;        // positions of a tile
    static constexpr int kChannels = kGroups * EPT;
};

template <int V, int EPT, int LC>
struct Shared {
    using S = Shape<V, EPT, LC>;
    float vec[kVectors][S::kChannels];
    float2 part[S::kGroups][S::kPos];
    float2 stat[S::kPos];
};

// The weights in fp32 with their defaults; zeros for channels past the last.
template <typename T, typename SH>
__device__ void load_vectors(SH& sh, const Problem& p, int channels) {
    for (int c = threadIdx.x; c < channels; c += blockDim.x) {
        const bool live = c < p.channels;
        sh.vec[kPostW][c] = live ? weight<T>(p.post_w, c, p.wide, 1.f) : 0.f;
        sh.vec[kPostB][c] = live ? weight<T>(p.post_b, c, p.wide, 0.f) : 0.f;
        sh.vec[kPreW][c] = live ? weight<T>(p.pre_w, c, p.wide, 1.f) : 0.f;
        sh.vec[kPreB][c] = live ? weight<T>(p.pre_b, c, p.wide, 0.f) : 0.f;
        sh.vec[kScaleW][c] = live ? p.scale * weight<T>(p.scale_w, c, p.wide, 1.f) : 0.f;
    }
    __syncthreads();
}

// Mean and 1 / sqrt(variance + eps) over the channels of each of a thread's V positions; `keep`
// (may be null) receives them per position.  Every thread of the block calls it.
template <int V, int EPT, int LC>
__device__ __forceinline__ void statistics(Shared<V, EPT, LC>& sh, const Problem& p, const float (&v)[EPT][V], int group,
                                           int groups, int pos, float (&mean)[V], float (&rho)[V], float* keep,
                                           int live_pos) {
    const int mine = max(0, min(EPT, p.channels - group * EPT));
#pragma unroll
    for (int i = 0; i < V; ++i) {
        float m = 0.f, s = 0.f;
        if (p.kind == kLayer) {
#pragma unroll
            for (int j = 0; j < EPT; ++j) m += j < mine ? v[j][i] : 0.f;
            m = mine ? m / static_cast<float>(mine) : 0.f;
        }
#pragma unroll
        for (int j = 0; j < EPT; ++j) {
            const float d = j < mine ? v[j][i] - m : 0.f;
            s = fmaf(d, d, s);
        }
        sh.part[group][pos * V + i] = make_float2(m, s);
    }
    __syncthreads();
    for (int q = threadIdx.x; q < Shape<V, EPT, LC>::kPos; q += blockDim.x) {
        float m = 0.f, s = 0.f;
        if (p.kind == kLayer) {
            for (int g = 0; g < groups; ++g)
                m = fmaf(static_cast<float>(max(0, min(EPT, p.channels - g * EPT))), sh.part[g][q].x, m);
            m *= p.inv_c;
            for (int g = 0; g < groups; ++g) {
                const float2 a = sh.part[g][q];
                const float d = a.x - m;
                s += fmaf(static_cast<float>(max(0, min(EPT, p.channels - g * EPT))) * d, d, a.y);
            }
        } else {
            for (int g = 0; g < groups; ++g) s += sh.part[g][q].y;
        }
        const float r = 1.f / sqrtf(fmaf(s, p.inv_c, p.eps));
        sh.stat[q] = make_float2(m, r);
        if (keep != nullptr && q < live_pos) {
            keep[q] = m;
            keep[p.positions + q] = r;
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const float2 a = sh.stat[pos * V + i];
        mean[i] = a.x;
        rho[i] = a.y;
    }
}

// Means over the channels of two products, per position; every thread of the block calls it.
template <int V, int EPT, int LC>
__device__ __forceinline__ void two_means(Shared<V, EPT, LC>& sh, const Problem& p, const float2 (&part)[V], int group,
                                          int groups, int pos, float2 (&mean)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) sh.part[group][pos * V + i] = part[i];
    __syncthreads();
    for (int q = threadIdx.x; q < Shape<V, EPT, LC>::kPos; q += blockDim.x) {
        float a = 0.f, b = 0.f;
        for (int g = 0; g < groups; ++g) {
            a += sh.part[g][q].x;
            b += sh.part[g][q].y;
        }
        sh.stat[q] = make_float2(p.kind == kLayer ? a * p.inv_c : 0.f, b * p.inv_c);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < V; ++i) mean[i] = sh.stat[pos * V + i];
}

struct Where {
    int group, groups, pos, c0;
};

template <int EPT, int LC>
__device__ __forceinline__ Where where() {
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int group = warp * LC + lane / (32 / LC);
    return {group, static_cast<int>(blockDim.x) / 32 * LC, lane % (32 / LC), group * EPT};
}

template <typename T, int V, int EPT, int LC>
__global__ void __launch_bounds__(kMaxWarps * 32) field_forward_kernel(const __grid_constant__ Problem p) {
    using S = Shape<V, EPT, LC>;
    __shared__ Shared<V, EPT, LC> sh;
    const Where at = where<EPT, LC>();
    load_vectors<T>(sh, p, at.groups * EPT);
    const int ts = static_cast<int>(p.tiles_per_sample);
    for (int tile = blockIdx.x; tile < static_cast<int>(p.tiles); tile += gridDim.x) {
        const int sample = tile / ts;
        const int l0 = (tile - sample * ts) * S::kPos;
        const long long l = l0 + at.pos * V;
        const size_t base = static_cast<size_t>(sample) * p.channels * p.length + l;
        const size_t q0 = static_cast<size_t>(sample) * p.length + l0;
        const int live_pos = static_cast<int>(min(static_cast<long long>(S::kPos), p.length - l0));
        const int end = l < p.length ? min(EPT, p.channels - at.c0) : 0;  // of this thread's channels
        Vec<T, V> x[EPT], y[EPT], g[EPT];
#pragma unroll
        for (int j = 0; j < EPT; ++j) {
            if (j < end) {
                const size_t e = base + static_cast<size_t>(at.c0 + j) * p.length;
                x[j] = load_vec<T, V>(p.x, e);
                if (p.y) y[j] = load_vec<T, V>(p.y, e);
                if (p.gate_mode == kGateFull) g[j] = load_vec<T, V>(p.gate, e);
            } else {
                x[j] = y[j] = g[j] = Vec<T, V>{};
            }
        }
        float r[EPT][V], mean[V], rho[V];
        if (p.y) {
            if (p.post) {
#pragma unroll
                for (int j = 0; j < EPT; ++j)
#pragma unroll
                    for (int i = 0; i < V; ++i) r[j][i] = to_f32(y[j].v[i]);
                statistics<V, EPT, LC>(sh, p, r, at.group, at.groups, at.pos, mean, rho, p.stats ? p.stats + q0 : nullptr,
                                       live_pos);
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) mean[i] = 0.f, rho[i] = 1.f;
            }
#pragma unroll
            for (int j = 0; j < EPT; ++j) {
                const float w = p.post ? sh.vec[kPostW][at.c0 + j] : 1.f, b = p.post ? sh.vec[kPostB][at.c0 + j] : 0.f;
                const float scale = sh.vec[kScaleW][at.c0 + j];
                float a = 1.f;
                if (p.gate_mode == kGateSample && j < end)
                    a = activate(to_f32(static_cast<const T*>(p.gate)[static_cast<size_t>(sample) * p.channels + at.c0 + j]),
                                 p.act);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    if (p.gate_mode == kGateFull) a = activate(to_f32(g[j].v[i]), p.act);
                    const float h = (to_f32(y[j].v[i]) - mean[i]) * rho[i];
                    r[j][i] = fmaf(scale * a, fmaf(h, w, b), to_f32(x[j].v[i]));
                }
                if (j < end) {
                    Vec<T, V> o;
#pragma unroll
                    for (int i = 0; i < V; ++i) from_f32(o.v[i], r[j][i]);
                    store_vec<T, V>(p.r, base + static_cast<size_t>(at.c0 + j) * p.length, o);
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < EPT; ++j)
#pragma unroll
                for (int i = 0; i < V; ++i) r[j][i] = to_f32(x[j].v[i]);
        }
        if (!p.pre) continue;
        statistics<V, EPT, LC>(sh, p, r, at.group, at.groups, at.pos, mean, rho,
                               p.stats ? p.stats + 2 * p.positions + q0 : nullptr, live_pos);
#pragma unroll
        for (int j = 0; j < EPT; ++j) {
            if (j >= end) continue;
            const float w = sh.vec[kPreW][at.c0 + j], b = sh.vec[kPreB][at.c0 + j];
            Vec<T, V> o;
#pragma unroll
            for (int i = 0; i < V; ++i) from_f32(o.v[i], fmaf((r[j][i] - mean[i]) * rho[i], w, b));
            store_vec<T, V>(p.n, base + static_cast<size_t>(at.c0 + j) * p.length, o);
        }
    }
}

// Adds v over the lanes that share this lane's channel group.
template <int LC>
__device__ __forceinline__ float sum_positions(float v) {
#pragma unroll
    for (int o = 16 / LC; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

template <typename T, int V, int EPT, int LC>
__global__ void __launch_bounds__(kMaxWarps * 32) field_backward_kernel(const __grid_constant__ Problem p) {
    using S = Shape<V, EPT, LC>;
    __shared__ Shared<V, EPT, LC> sh;
    grid_dep_launch();
    const Where at = where<EPT, LC>();
    load_vectors<T>(sh, p, at.groups * EPT);
    const long long last = tile_begin(p, blockIdx.x + 1);
    float sum[kSums][EPT] = {};
    for (long long tile = tile_begin(p, blockIdx.x); tile < last; ++tile) {
        const int sample = static_cast<int>(tile) / static_cast<int>(p.tiles_per_sample);
        const long long l = (tile - sample * p.tiles_per_sample) * S::kPos + at.pos * V;
        const size_t base = static_cast<size_t>(sample) * p.channels * p.length + l;
        const int end = l < p.length ? min(EPT, p.channels - at.c0) : 0;
        Vec<T, V> x[EPT], y[EPT], g[EPT], dr[EPT], dn[EPT];
#pragma unroll
        for (int j = 0; j < EPT; ++j) {
            x[j] = y[j] = g[j] = dr[j] = dn[j] = Vec<T, V>{};
            if (j < end) {
                const size_t e = base + static_cast<size_t>(at.c0 + j) * p.length;
                if (p.dn) dn[j] = load_vec<T, V>(p.dn, e);
                if (p.y) y[j] = load_vec<T, V>(p.y, e);
                if (p.dn) x[j] = load_vec<T, V>(p.x, e);
                if (p.gate_mode == kGateFull) g[j] = load_vec<T, V>(p.gate, e);
                if (p.dr) dr[j] = load_vec<T, V>(p.dr, e);
            }
        }
        Vec<float, V> mean{}, rho{}, mean2{}, rho2{};
        if (end > 0) {
            const float* st = p.stats + static_cast<size_t>(sample) * p.length + l;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                mean.v[i] = p.post ? st[i] : 0.f;
                rho.v[i] = p.post ? st[p.positions + i] : 1.f;
                mean2.v[i] = p.pre ? st[2 * p.positions + i] : 0.f;
                rho2.v[i] = p.pre ? st[3 * p.positions + i] : 0.f;
            }
        }
        // act(gate) of the thread's channels: per element in full mode, per channel otherwise
        float a[EPT][V], slope[EPT][V];
#pragma unroll
        for (int j = 0; j < EPT; ++j) {
            float one = 1.f;
            if (p.gate_mode == kGateSample && j < end)
                one = activate(to_f32(static_cast<const T*>(p.gate)[static_cast<size_t>(sample) * p.channels + at.c0 + j]),
                               p.act);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                a[j][i] = one;
                slope[j][i] = 0.f;
                if (p.gate_mode == kGateFull) a[j][i] = activate(to_f32(g[j].v[i]), p.act, slope[j][i]);
            }
        }
        float h[EPT][V], k[EPT][V], t[EPT][V];
        float2 m[V];
#pragma unroll
        for (int i = 0; i < V; ++i) m[i] = make_float2(0.f, 0.f);
#pragma unroll
        for (int j = 0; j < EPT; ++j) {
            const float w = p.post ? sh.vec[kPostW][at.c0 + j] : 1.f, b = p.post ? sh.vec[kPostB][at.c0 + j] : 0.f;
            const float scale = sh.vec[kScaleW][at.c0 + j], w2 = sh.vec[kPreW][at.c0 + j];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                h[j][i] = p.y ? (to_f32(y[j].v[i]) - mean.v[i]) * rho.v[i] : 0.f;
                const float r = fmaf(scale * a[j][i], fmaf(h[j][i], w, b), to_f32(x[j].v[i]));
                k[j][i] = (r - mean2.v[i]) * rho2.v[i];
                const float d = to_f32(dn[j].v[i]) * w2;
                t[j][i] = d;
                if (j < end) {
                    m[i].x += d;
                    m[i].y = fmaf(d, k[j][i], m[i].y);
                    sum[kDPreW][j] = fmaf(to_f32(dn[j].v[i]), k[j][i], sum[kDPreW][j]);
                    sum[kDPreB][j] += to_f32(dn[j].v[i]);
                }
            }
        }
        if (p.dn) two_means<V, EPT, LC>(sh, p, m, at.group, at.groups, at.pos, m);
        float2 m2[V];
#pragma unroll
        for (int i = 0; i < V; ++i) m2[i] = make_float2(0.f, 0.f);
#pragma unroll
        for (int j = 0; j < EPT; ++j) {
            const float ws = (p.post ? sh.vec[kPostW][at.c0 + j] : 1.f) * sh.vec[kScaleW][at.c0 + j];
            Vec<T, V> o;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                t[j][i] = to_f32(dr[j].v[i]) + rho2.v[i] * (t[j][i] - m[i].x - k[j][i] * m[i].y);
                from_f32(o.v[i], t[j][i]);
                if (j < end) {
                    const float d = t[j][i] * a[j][i] * ws;
                    m2[i].x += d;
                    m2[i].y = fmaf(d, h[j][i], m2[i].y);
                    const float ta = p.slots ? t[j][i] : t[j][i] * a[j][i];
                    sum[kTah][j] = fmaf(ta, h[j][i], sum[kTah][j]);
                    sum[kTa][j] += ta;
                }
            }
            if (p.dx && j < end) store_vec<T, V>(p.dx, base + static_cast<size_t>(at.c0 + j) * p.length, o);
        }
        if (p.post && p.dy) two_means<V, EPT, LC>(sh, p, m2, at.group, at.groups, at.pos, m2);
#pragma unroll
        for (int j = 0; j < EPT; ++j) {
            if (j >= end) continue;
            const size_t e = base + static_cast<size_t>(at.c0 + j) * p.length;
            const float w = p.post ? sh.vec[kPostW][at.c0 + j] : 1.f, b = p.post ? sh.vec[kPostB][at.c0 + j] : 0.f;
            const float scale = sh.vec[kScaleW][at.c0 + j];
            Vec<T, V> o;
            if (p.dy) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float d = t[j][i] * a[j][i] * (scale * w);
                    from_f32(o.v[i], p.post ? rho.v[i] * (d - m2[i].x - h[j][i] * m2[i].y) : d);
                }
                store_vec<T, V>(p.dy, e, o);
            }
            if (p.dgate && p.gate_mode == kGateFull) {
#pragma unroll
                for (int i = 0; i < V; ++i) from_f32(o.v[i], t[j][i] * scale * fmaf(h[j][i], w, b) * slope[j][i]);
                store_vec<T, V>(p.dgate, e, o);
            }
        }
        if (p.slots && (tile + 1 == last || (tile + 1) % p.tiles_per_sample == 0)) {
            float* slot = slot_of(p, blockIdx.x, sample);
#pragma unroll
            for (int j = 0; j < EPT; ++j) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float total = sum_positions<LC>(sum[kTah + i][j]);
                    if (at.pos == 0 && at.c0 + j < p.channels)
                        slot[static_cast<size_t>(i) * p.channels + at.c0 + j] = total;
                    sum[kTah + i][j] = 0.f;
                }
            }
        }
    }
    if (!p.sums) return;
#pragma unroll
    for (int i = 0; i < kSums; ++i) {
#pragma unroll
        for (int j = 0; j < EPT; ++j) {
            const float total = sum_positions<LC>(sum[i][j]);
            if (at.pos == 0 && at.c0 + j < p.channels)
                p.partial[(static_cast<size_t>(blockIdx.x) * kSums + i) * p.channels + at.c0 + j] = total;
        }
    }
}

// Sets the tiles of a shape; false where it has more than 32 bits count.
template <typename S>
bool tile(Problem& p) {
    p.tiles_per_sample = (p.length + S::kPos - 1) / S::kPos;
    p.tiles = p.batch * p.tiles_per_sample;
    return p.tiles < (1LL << 30) && p.length < (1LL << 30);
}

template <int EPT, int LC>
int threads_for(int channels) {
    return (channels + EPT * LC - 1) / (EPT * LC) * 32;
}

template <typename T, int V, int EPT, int LC>
cudaError_t forward_as(Problem p, cudaStream_t s) {
    if (!tile<Shape<V, EPT, LC>>(p)) return cudaErrorNotSupported;
    const int threads = threads_for<EPT, LC>(p.channels);
    int per_sm = 0;
    const cudaError_t e =
        scx::prepare_kernel(reinterpret_cast<const void*>(field_forward_kernel<T, V, EPT, LC>), 0, threads, &per_sm);
    if (e != cudaSuccess) return e;
    const int grid = static_cast<int>(std::min<long long>(p.tiles, 4LL * per_sm * scx::num_sms()));
    field_forward_kernel<T, V, EPT, LC><<<grid, threads, 0, s>>>(p);
    return cudaGetLastError();
}

template <typename T, int V, int EPT, int LC>
cudaError_t backward_as(Problem& p, cudaStream_t s) {
    Problem q = p;
    if (!tile<Shape<V, EPT, LC>>(q)) return cudaErrorNotSupported;
    const int threads = threads_for<EPT, LC>(p.channels);
    int per_sm = 0;
    const cudaError_t e =
        scx::prepare_kernel(reinterpret_cast<const void*>(field_backward_kernel<T, V, EPT, LC>), 0, threads, &per_sm);
    if (e != cudaSuccess) return e;
    q.parts = static_cast<int>(
        std::min<long long>(std::min(max_parts(p.channels), per_sm * scx::num_sms()), q.tiles));
    p = q;
    field_backward_kernel<T, V, EPT, LC><<<p.parts, threads, 0, s>>>(p);
    return cudaGetLastError();
}

// Whether V positions can be moved by one access: rows of a multiple of V, every base aligned.
template <typename T, int V>
bool vectors_fit(const Problem& p) {
    const void* all[] = {p.x, p.y, p.gate_mode == kGateFull ? p.gate : nullptr, p.r, p.n, p.dr, p.dn, p.dx, p.dy,
                         p.gate_mode == kGateFull ? p.dgate : nullptr};
    for (const void* a : all)
        if (!aligned(a, V * sizeof(T))) return false;
    return p.length % V == 0;
}

}  // namespace

template <typename T>
cudaError_t field_forward(const Problem& p, cudaStream_t s) {
    if (p.channels <= 4 * kMaxWarps) {
        if (vectors_fit<T, 4>(p)) return forward_as<T, 4, 4, 1>(p, s);
        return forward_as<T, 1, 4, 1>(p, s);
    }
    if (p.channels <= 8 * kMaxWarps) {
        if (vectors_fit<T, 2>(p)) return forward_as<T, 2, 8, 1>(p, s);
        return forward_as<T, 1, 8, 1>(p, s);
    }
    if (p.channels <= 32 * kMaxWarps) return forward_as<T, 1, 8, 4>(p, s);
    return cudaErrorNotSupported;
}

template <typename T>
cudaError_t field_backward(Problem& p, cudaStream_t s) {
    if (p.channels <= 4 * kMaxWarps) {
        if (vectors_fit<T, 2>(p)) return backward_as<T, 2, 4, 1>(p, s);
        return backward_as<T, 1, 4, 1>(p, s);
    }
    if (p.channels <= 8 * kMaxWarps) return backward_as<T, 1, 8, 1>(p, s);
    if (p.channels <= 32 * kMaxWarps) return backward_as<T, 1, 8, 4>(p, s);
    return cudaErrorNotSupported;
}

template cudaError_t field_forward<float>(const Problem&, cudaStream_t);
template cudaError_t field_forward<__nv_bfloat16>(const Problem&, cudaStream_t);
template cudaError_t field_forward<__half>(const Problem&, cudaStream_t);
template cudaError_t field_backward<float>(Problem&, cudaStream_t);
template cudaError_t field_backward<__nv_bfloat16>(Problem&, cudaStream_t);
template cudaError_t field_backward<__half>(Problem&, cudaStream_t);

}  // namespace scx_rn
