// The residual-norm kernels for fields, [batch][channels][length]: a position's channels lie
// `length` elements apart, so a warp takes neighbouring positions of a few channels, and a block's
// warps together all channels of a tile of positions.
//
// A thread has V neighbouring positions (one access) of kEpt channels, and every tensor is read
// once: the next tile's values are copied into the thread's own slots in shared memory while this
// tile's are in registers.  A warp's 32 lanes are 32/LC positions x LC channel groups; LC > 1
// serves channel counts that would take more than 16 warps.  A statistic is a sum over a
// position's channel groups: each group leaves its part in shared memory, one thread per position
// adds them and leaves the result.  The layer kind's variance is not taken from sums of squares: a
// group leaves its mean and its sum of squares about it, and the parts are joined about the common
// mean.
#pragma once

#include <algorithm>

#include "scx_internal.h"
#include "scx_residual_norm.cuh"

namespace scx_rn {
namespace {

constexpr int kMaxWarps = 16;
constexpr int kEpt = 4;  // channels per thread
enum : int { kPostW = 0, kPostB = 1, kPreW = 2, kPreB = 3, kVectors = 4 };

template <int V, int LC>
struct Shape {
    static constexpr int kGroups = kMaxWarps * LC;  // most channel groups of a block
    static constexpr int kPos = 32 / LC * V;        // positions of a tile
    static constexpr int kChannels = kGroups * kEpt;
};

template <int V, int LC>
struct alignas(16) Shared {
    using S = Shape<V, LC>;
    float vec[kVectors][S::kChannels];
    float2 part[S::kGroups][S::kPos];
    float2 stat[S::kPos];
};

// The weights in fp32 with their defaults, the scale taken into those of the norm after the block;
// zeros for channels past the last.
template <typename T, typename SH>
__device__ void load_vectors(SH& sh, const Problem& p, int channels) {
    for (int c = threadIdx.x; c < channels; c += blockDim.x) {
        const bool live = c < p.channels;
        const float scale = live ? p.scale * weight<T>(p.scale_w, c, p.wide, 1.f) : 0.f;
        sh.vec[kPostW][c] = live ? scale * (p.post ? weight<T>(p.post_w, c, p.wide, 1.f) : 1.f) : 0.f;
        sh.vec[kPostB][c] = live ? scale * (p.post ? weight<T>(p.post_b, c, p.wide, 0.f) : 0.f) : 0.f;
        sh.vec[kPreW][c] = live ? weight<T>(p.pre_w, c, p.wide, 1.f) : 0.f;
        sh.vec[kPreB][c] = live ? weight<T>(p.pre_b, c, p.wide, 0.f) : 0.f;
    }
    __syncthreads();
}

struct Where {
    int group, groups, pos, c0, mine;  // mine: the thread's channels that exist
};

template <int LC>
__device__ __forceinline__ Where where(const Problem& p) {
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int group = warp * LC + lane / (32 / LC);
    return {group, static_cast<int>(blockDim.x) / 32 * LC, lane % (32 / LC), group * kEpt,
            max(0, min(kEpt, p.channels - group * kEpt))};
}

// Mean and 1 / sqrt(variance + eps) over the channels of each of a thread's V positions; `keep`
// (may be null) receives them per position.  Every thread of the block calls it.
template <int V, int LC>
__device__ __forceinline__ void statistics(Shared<V, LC>& sh, const Problem& p, const float (&v)[kEpt * V],
                                           const Where& at, float (&mean)[V], float (&rho)[V], float* keep,
                                           int live_pos) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
        float m = 0.f, s = 0.f;
        if (p.kind == kLayer) {  // channels that do not exist hold zeros
#pragma unroll
            for (int j = 0; j < kEpt; ++j) m += v[j * V + i];
            m = at.mine ? m / static_cast<float>(at.mine) : 0.f;
#pragma unroll
            for (int j = 0; j < kEpt; ++j) {
                const float d = j < at.mine ? v[j * V + i] - m : 0.f;
                s = fmaf(d, d, s);
            }
        } else {
#pragma unroll
            for (int j = 0; j < kEpt; ++j) s = fmaf(v[j * V + i], v[j * V + i], s);
        }
        sh.part[at.group][at.pos * V + i] = make_float2(m, s);
    }
    __syncthreads();
    for (int q = threadIdx.x; q < Shape<V, LC>::kPos; q += blockDim.x) {
        float m = 0.f, s = 0.f;
        if (p.kind == kLayer) {
            for (int g = 0; g < at.groups; ++g)
                m = fmaf(static_cast<float>(max(0, min(kEpt, p.channels - g * kEpt))), sh.part[g][q].x, m);
            m *= p.inv_c;
            for (int g = 0; g < at.groups; ++g) {
                const float2 a = sh.part[g][q];
                const float d = a.x - m;
                s += fmaf(static_cast<float>(max(0, min(kEpt, p.channels - g * kEpt))) * d, d, a.y);
            }
        } else {
#pragma unroll 4
            for (int g = 0; g < at.groups; ++g) s += sh.part[g][q].y;
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
        const float2 a = sh.stat[at.pos * V + i];
        mean[i] = a.x;
        rho[i] = a.y;
    }
}

// Means over the channels of two products, per position; every thread of the block calls it.
template <int V, int LC>
__device__ __forceinline__ void two_means(Shared<V, LC>& sh, const Problem& p, const Where& at, float2 (&mean)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) sh.part[at.group][at.pos * V + i] = mean[i];
    __syncthreads();
    for (int q = threadIdx.x; q < Shape<V, LC>::kPos; q += blockDim.x) {
        float a = 0.f, b = 0.f;
#pragma unroll 4
        for (int g = 0; g < at.groups; ++g) {
            a += sh.part[g][q].x;
            b += sh.part[g][q].y;
        }
        sh.stat[q] = make_float2(p.kind == kLayer ? a * p.inv_c : 0.f, b * p.inv_c);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < V; ++i) mean[i] = sh.stat[at.pos * V + i];
}

// Where a tile lies, for one thread.
template <int V, int LC>
struct Tile {
    int sample, l0;
    bool live;    // whether the thread's positions exist
    size_t base;  // the thread's first element

    __device__ __forceinline__ Tile(const Problem& p, const Where& at, int tile) {
        const int ts = static_cast<int>(p.tiles_per_sample);
        sample = tile / ts;
        l0 = (tile - sample * ts) * Shape<V, LC>::kPos;
        const int l = l0 + at.pos * V;
        live = l < static_cast<int>(p.length);
        base = (static_cast<size_t>(sample) * p.channels + at.c0) * p.length + l;
    }
};

// A thread's slots for one tensor of one tile, and how it fills and reads them.
template <typename T, int V>
struct Slots {
    using E = Vec<T, V>;

    static __device__ __forceinline__ void fetch(E* slot, const void* from, size_t base, size_t stride, int end) {
        if constexpr (kCopied<E>) {
#pragma unroll
            for (int j = 0; j < kEpt; ++j)
                copy_async(slot + j * blockDim.x, static_cast<const T*>(from) + (j < end ? base + j * stride : 0), j < end);
        }
    }

    static __device__ __forceinline__ void read(const E* slot, const void* from, size_t base, size_t stride, int end,
                                                float (&out)[kEpt * V]) {
#pragma unroll
        for (int j = 0; j < kEpt; ++j) {
            E v{};
            if constexpr (kCopied<E>) v = slot[j * blockDim.x];
            else if (j < end) v = load_vec<T, V>(from, base + j * stride);
#pragma unroll
            for (int i = 0; i < V; ++i) out[j * V + i] = to_f32(v.v[i]);
        }
    }
};

template <typename T, int V>
__device__ __forceinline__ void store_all(void* to, size_t base, size_t stride, int end, const float (&v)[kEpt * V]) {
#pragma unroll
    for (int j = 0; j < kEpt; ++j) {
        Vec<T, V> o;
#pragma unroll
        for (int i = 0; i < V; ++i) from_f32(o.v[i], v[j * V + i]);
        if (j < end) store_vec<T, V>(to, base + j * stride, o);
    }
}

// act(gate) of a thread's channels, the gate being one value per sample and channel.
template <typename T, int V>
__device__ __forceinline__ void sample_gate(const Problem& p, const Where& at, int sample, float (&a)[kEpt * V]) {
    float g[kEpt];
#pragma unroll
    for (int j = 0; j < kEpt; ++j)
        g[j] = j < at.mine ? to_f32(static_cast<const T*>(p.gate)[static_cast<size_t>(sample) * p.channels + at.c0 + j]) : 0.f;
    activate_all(g, p.act);
#pragma unroll
    for (int j = 0; j < kEpt; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) a[j * V + i] = g[j];
}

__host__ __device__ constexpr int forward_tensors(int mode) { return mode == kNoBlock ? 1 : mode == kFull ? 3 : 2; }

template <typename T, int V, int LC, int MODE>
__global__ void __launch_bounds__(kMaxWarps * 32, 2) field_forward_kernel(const __grid_constant__ Problem p) {
    using S = Shape<V, LC>;
    using F = Slots<T, V>;
    extern __shared__ __align__(16) unsigned char dynamic[];
    auto& sh = *reinterpret_cast<Shared<V, LC>*>(dynamic);
    const Where at = where<LC>(p);
    const size_t stride = static_cast<size_t>(p.length);
    const int tiles = static_cast<int>(p.tiles);
    constexpr int kTensors = forward_tensors(MODE);
    auto* slots = reinterpret_cast<typename F::E*>(dynamic + sizeof(sh)) + threadIdx.x;
    auto slot = [&](int turn, int tensor) { return slots + (turn * kTensors + tensor) * kEpt * blockDim.x; };
    auto fetch = [&](int tile, int turn) {
        if (tile < tiles) {
            const Tile<V, LC> t(p, at, tile);
            const int end = t.live ? at.mine : 0;
            F::fetch(slot(turn, 0), p.x, t.base, stride, end);
            if constexpr (MODE != kNoBlock) F::fetch(slot(turn, 1), p.y, t.base, stride, end);
            if constexpr (MODE == kFull) F::fetch(slot(turn, 2), p.gate, t.base, stride, end);
        }
        copy_commit();
    };
    fetch(blockIdx.x, 0);
    load_vectors<T>(sh, p, at.groups * kEpt);
    int turn = 0;
    for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x, turn ^= 1) {
        const Tile<V, LC> t(p, at, tile);
        const int end = t.live ? at.mine : 0;
        const size_t q0 = static_cast<size_t>(t.sample) * p.length + t.l0;
        const int live_pos = min(S::kPos, static_cast<int>(p.length) - t.l0);
        fetch(tile + gridDim.x, turn ^ 1);
        copy_wait<1>();
        float r[kEpt * V], mean[V], rho[V];
        F::read(slot(turn, 0), p.x, t.base, stride, end, r);
        if constexpr (MODE != kNoBlock) {
            float h[kEpt * V], a[kEpt * V];
            F::read(slot(turn, 1), p.y, t.base, stride, end, h);
            if constexpr (MODE == kFull) F::read(slot(turn, 2), p.gate, t.base, stride, end, a);
            if (p.post) {
                statistics<V, LC>(sh, p, h, at, mean, rho, p.stats ? p.stats + q0 : nullptr, live_pos);
#pragma unroll
                for (int j = 0; j < kEpt * V; ++j) h[j] = (h[j] - mean[j % V]) * rho[j % V];
            }
            if constexpr (MODE == kFull) activate_all(a, p.act);
            if constexpr (MODE == kSample) sample_gate<T, V>(p, at, t.sample, a);
#pragma unroll
            for (int j = 0; j < kEpt; ++j) {
                const float w = sh.vec[kPostW][at.c0 + j], b = sh.vec[kPostB][at.c0 + j];
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float z = fmaf(h[j * V + i], w, b);
                    r[j * V + i] = MODE == kPlain ? r[j * V + i] + z : fmaf(a[j * V + i], z, r[j * V + i]);
                }
            }
            store_all<T, V>(p.r, t.base, stride, end, r);
        }
        if (!p.pre) continue;
        statistics<V, LC>(sh, p, r, at, mean, rho, p.stats ? p.stats + 2 * p.positions + q0 : nullptr, live_pos);
#pragma unroll
        for (int j = 0; j < kEpt; ++j) {
            const float w = sh.vec[kPreW][at.c0 + j], b = sh.vec[kPreB][at.c0 + j];
#pragma unroll
            for (int i = 0; i < V; ++i) r[j * V + i] = fmaf((r[j * V + i] - mean[i]) * rho[i], w, b);
        }
        store_all<T, V>(p.n, t.base, stride, end, r);
    }
    copy_wait<0>();
}

// Adds v over the lanes that share this lane's channel group.
template <int LC>
__device__ __forceinline__ float sum_positions(float v) {
#pragma unroll
    for (int o = 16 / LC; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Tensors a backward reads: x, y, dn, dr, and a gate per element.
__host__ __device__ constexpr int backward_tensors(int mode) { return mode == kFull ? 5 : 4; }

template <typename T, int V, int LC, int MODE>
__global__ void __launch_bounds__(kMaxWarps * 32) field_backward_kernel(const __grid_constant__ Problem p) {
    using F = Slots<T, V>;
    constexpr int N = kEpt * V;
    extern __shared__ __align__(16) unsigned char dynamic[];
    auto& sh = *reinterpret_cast<Shared<V, LC>*>(dynamic);
    grid_dep_launch();
    const Where at = where<LC>(p);
    const size_t stride = static_cast<size_t>(p.length);
    constexpr int kTensors = backward_tensors(MODE);
    auto* slots = reinterpret_cast<typename F::E*>(dynamic + sizeof(sh)) + threadIdx.x;
    auto slot = [&](int turn, int tensor) { return slots + (turn * kTensors + tensor) * kEpt * blockDim.x; };
    const int first = static_cast<int>(tile_begin(p, blockIdx.x)), last = static_cast<int>(tile_begin(p, blockIdx.x + 1));
    auto fetch = [&](int tile, int turn) {
        if (tile < last) {
            const Tile<V, LC> t(p, at, tile);
            const int end = t.live ? at.mine : 0;
            if constexpr (MODE != kNoBlock) F::fetch(slot(turn, 1), p.y, t.base, stride, end);
            if (p.dn) {
                F::fetch(slot(turn, 0), p.x, t.base, stride, end);
                F::fetch(slot(turn, 2), p.dn, t.base, stride, end);
            }
            if (p.dr) F::fetch(slot(turn, 3), p.dr, t.base, stride, end);
            if constexpr (MODE == kFull) F::fetch(slot(turn, 4), p.gate, t.base, stride, end);
        }
        copy_commit();
    };
    fetch(first, 0);
    load_vectors<T>(sh, p, at.groups * kEpt);
    int turn = 0;
    float sum[kSums][kEpt] = {};
    for (int tile = first; tile < last; ++tile, turn ^= 1) {
        const Tile<V, LC> t(p, at, tile);
        const int end = t.live ? at.mine : 0;
        float mean[V], rho[V], mean2[V], rho2[V];
        {
            const float* st = p.stats + static_cast<size_t>(t.sample) * p.length + t.l0 + at.pos * V;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                mean[i] = t.live && p.post ? st[i] : 0.f;
                rho[i] = t.live ? (p.post ? st[p.positions + i] : 1.f) : 0.f;
                mean2[i] = t.live && p.dn ? st[2 * p.positions + i] : 0.f;
                rho2[i] = t.live && p.dn ? st[3 * p.positions + i] : 0.f;
            }
        }
        fetch(tile + 1, turn ^ 1);
        copy_wait<1>();
        float h[N], a[N], slope[N], k[N], g[N];
        if constexpr (MODE != kNoBlock) {
            F::read(slot(turn, 1), p.y, t.base, stride, end, h);
#pragma unroll
            for (int j = 0; j < N; ++j) h[j] = (h[j] - mean[j % V]) * rho[j % V];
            if constexpr (MODE == kFull) {
                F::read(slot(turn, 4), p.gate, t.base, stride, end, a);
                activate_all(a, slope, p.act);
            }
            if constexpr (MODE == kSample) sample_gate<T, V>(p, at, t.sample, a);
        }
        float2 m[V];
#pragma unroll
        for (int i = 0; i < V; ++i) m[i] = make_float2(0.f, 0.f);
        if (p.dn) {
            F::read(slot(turn, 0), p.x, t.base, stride, end, k);
            F::read(slot(turn, 2), p.dn, t.base, stride, end, g);
#pragma unroll
            for (int j = 0; j < kEpt; ++j) {
                const float w = sh.vec[kPostW][at.c0 + j], b = sh.vec[kPostB][at.c0 + j], w2 = sh.vec[kPreW][at.c0 + j];
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const int e = j * V + i;
                    if constexpr (MODE != kNoBlock) {
                        const float z = fmaf(h[e], w, b);
                        k[e] = MODE == kPlain ? k[e] + z : fmaf(a[e], z, k[e]);
                    }
                    k[e] = (k[e] - mean2[i]) * rho2[i];
                    sum[kDPreW][j] = fmaf(g[e], k[e], sum[kDPreW][j]);
                    sum[kDPreB][j] += g[e];
                    g[e] *= w2;
                    m[i].x += g[e];
                    m[i].y = fmaf(g[e], k[e], m[i].y);
                }
            }
            two_means<V, LC>(sh, p, at, m);
#pragma unroll
            for (int e = 0; e < N; ++e) g[e] = rho2[e % V] * (g[e] - m[e % V].x - k[e] * m[e % V].y);
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e) g[e] = 0.f;
        }
        if (p.dr) {
            F::read(slot(turn, 3), p.dr, t.base, stride, end, k);
#pragma unroll
            for (int e = 0; e < N; ++e) g[e] += k[e];
        }
        // g: the gradient of r
        if (p.dx) store_all<T, V>(p.dx, t.base, stride, end, g);
        if constexpr (MODE != kNoBlock) {
#pragma unroll
            for (int i = 0; i < V; ++i) m[i] = make_float2(0.f, 0.f);
#pragma unroll
            for (int j = 0; j < kEpt; ++j) {
                const float w = sh.vec[kPostW][at.c0 + j];
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const int e = j * V + i;
                    const float ta = MODE == kPlain ? g[e] : g[e] * a[e];
                    const float v = MODE == kSample ? g[e] : ta;
                    sum[kTah][j] = fmaf(v, h[e], sum[kTah][j]);
                    sum[kTa][j] += v;
                    k[e] = ta * w;
                    m[i].x += k[e];
                    m[i].y = fmaf(k[e], h[e], m[i].y);
                }
            }
            if (MODE == kFull && p.dgate) {
                float o[N];
#pragma unroll
                for (int j = 0; j < kEpt; ++j) {
                    const float w = sh.vec[kPostW][at.c0 + j], b = sh.vec[kPostB][at.c0 + j];
#pragma unroll
                    for (int i = 0; i < V; ++i)
                        o[j * V + i] = g[j * V + i] * fmaf(h[j * V + i], w, b) * slope[j * V + i];
                }
                store_all<T, V>(p.dgate, t.base, stride, end, o);
            }
            if (p.dy) {
                if (p.post) {
                    two_means<V, LC>(sh, p, at, m);
#pragma unroll
                    for (int e = 0; e < N; ++e) k[e] = rho[e % V] * (k[e] - m[e % V].x - h[e] * m[e % V].y);
                }
                store_all<T, V>(p.dy, t.base, stride, end, k);
            }
            if (MODE == kSample && p.slots &&
                (tile + 1 == last || t.l0 + Shape<V, LC>::kPos >= static_cast<int>(p.length))) {
                float* to = slot_of(p, blockIdx.x, t.sample);
#pragma unroll
                for (int j = 0; j < kEpt; ++j) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float total = sum_positions<LC>(sum[kTah + i][j]);
                        if (at.pos == 0 && j < at.mine) to[static_cast<size_t>(i) * p.channels + at.c0 + j] = total;
                        sum[kTah + i][j] = 0.f;
                    }
                }
            }
        }
    }
    copy_wait<0>();
    if (!p.sums) return;
#pragma unroll
    for (int i = 0; i < kSums; ++i) {
#pragma unroll
        for (int j = 0; j < kEpt; ++j) {
            const float total = sum_positions<LC>(sum[i][j]);
            if (at.pos == 0 && j < at.mine)
                p.partial[(static_cast<size_t>(blockIdx.x) * kSums + i) * p.channels + at.c0 + j] = total;
        }
    }
}

// Sets the tiles of a shape; false where their count or a position does not fit the kernels' int.
template <int V, int LC>
bool set_tiles(Problem& p) {
    constexpr int kPos = Shape<V, LC>::kPos;
    p.tiles_per_sample = (p.length + kPos - 1) / kPos;
    p.tiles = p.batch * p.tiles_per_sample;
    return p.tiles < (1LL << 30) && p.length < (1LL << 30);
}

template <int LC>
int threads_for(int channels) {
    return (channels + kEpt * LC - 1) / (kEpt * LC) * 32;
}

template <typename T, int V, int LC, int MODE>
cudaError_t forward_as(Problem p, cudaStream_t s) {
    if (!set_tiles<V, LC>(p)) return cudaErrorNotSupported;
    const int threads = threads_for<LC>(p.channels);
    const size_t smem = sizeof(Shared<V, LC>) +
                        (kCopied<Vec<T, V>> ? 2 * forward_tensors(MODE) * kEpt * sizeof(Vec<T, V>) * threads : 0);
    int per_sm = 0;
    const cudaError_t e =
        scx::prepare_kernel(reinterpret_cast<const void*>(field_forward_kernel<T, V, LC, MODE>), smem, threads, &per_sm);
    if (e != cudaSuccess) return e;
    const int grid = static_cast<int>(std::min<long long>(p.tiles, static_cast<long long>(per_sm) * scx::num_sms()));
    field_forward_kernel<T, V, LC, MODE><<<grid, threads, smem, s>>>(p);
    return cudaGetLastError();
}

template <typename T, int V, int LC, int MODE>
cudaError_t backward_as(Problem& p, cudaStream_t s) {
    Problem q = p;
    if (!set_tiles<V, LC>(q)) return cudaErrorNotSupported;
    const int threads = threads_for<LC>(p.channels);
    const size_t smem = sizeof(Shared<V, LC>) +
                        (kCopied<Vec<T, V>> ? 2 * backward_tensors(MODE) * kEpt * sizeof(Vec<T, V>) * threads : 0);
    int per_sm = 0;
    const cudaError_t e =
        scx::prepare_kernel(reinterpret_cast<const void*>(field_backward_kernel<T, V, LC, MODE>), smem, threads, &per_sm);
    if (e != cudaSuccess) return e;
    q.parts = static_cast<int>(std::min<long long>(std::min(max_parts(p.channels), per_sm * scx::num_sms()), q.tiles));
    p = q;
    field_backward_kernel<T, V, LC, MODE><<<p.parts, threads, smem, s>>>(p);
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

template <typename T, int MODE>
cudaError_t forward_in(const Problem& p, cudaStream_t s) {
    constexpr int kPer = kEpt * kMaxWarps;  // channels of a block at LC = 1
    if (vectors_fit<T, 2>(p)) {
        if (p.channels <= kPer) return forward_as<T, 2, 1, MODE>(p, s);
        if (p.channels <= 2 * kPer) return forward_as<T, 2, 2, MODE>(p, s);
        if (p.channels <= 8 * kPer) return forward_as<T, 2, 8, MODE>(p, s);
        return cudaErrorNotSupported;
    }
    if (p.channels <= kPer) return forward_as<T, 1, 1, MODE>(p, s);
    if (p.channels <= 4 * kPer) return forward_as<T, 1, 4, MODE>(p, s);
    return cudaErrorNotSupported;
}

template <typename T, int MODE>
cudaError_t backward_in(Problem& p, cudaStream_t s) {
    constexpr int kPer = kEpt * kMaxWarps;
    if (vectors_fit<T, 2>(p)) {
        if (p.channels <= kPer) return backward_as<T, 2, 1, MODE>(p, s);
        if (p.channels <= 2 * kPer) return backward_as<T, 2, 2, MODE>(p, s);
        if (p.channels <= 8 * kPer) return backward_as<T, 2, 8, MODE>(p, s);
        return cudaErrorNotSupported;
    }
    if (p.channels <= kPer) return backward_as<T, 1, 1, MODE>(p, s);
    if (p.channels <= 4 * kPer) return backward_as<T, 1, 4, MODE>(p, s);
    return cudaErrorNotSupported;
}

}  // namespace

template <typename T>
cudaError_t field_forward(const Problem& p, cudaStream_t s) {
    switch (mode_of(p)) {
        case kNoBlock: return forward_in<T, kNoBlock>(p, s);
        case kPlain: return forward_in<T, kPlain>(p, s);
        case kSample: return forward_in<T, kSample>(p, s);
        default: return forward_in<T, kFull>(p, s);
    }
}

template <typename T>
cudaError_t field_backward(Problem& p, cudaStream_t s) {
    switch (mode_of(p)) {
        case kNoBlock: return backward_in<T, kNoBlock>(p, s);
        case kPlain: return backward_in<T, kPlain>(p, s);
        case kSample: return backward_in<T, kSample>(p, s);
        default: return backward_in<T, kFull>(p, s);
    }
}

}  // namespace scx_rn
