// The residual-norm kernels for fields, [batch][channels][length]: a position's channels lie
// `length` elements apart, so a warp takes neighbouring positions of a few channels, and a block's
// warps together all channels of a tile of positions.
//
// A thread has V neighbouring positions (one access) of EPT channels, 8 values, and every
// tensor is read once: the next tile's values are copied into the thread's own slots in shared
// memory while this tile's are in registers.  A warp's 32 lanes are 32/LC positions x LC channel
// groups: LC = 2 keeps accesses of 16 bytes and warps of 4 channels, larger LC serves channel counts
// that would take more than 16 warps.  A statistic is a sum over a position's channels: within the
// thread, over the warp's channel groups by shuffles, and over the warps through shared memory,
// where a few threads per position add the warps' parts.  The layer kind's variance is not taken from
// sums of squares: a warp leaves its mean and its sum of squares about it, and the parts are joined
// about the common mean.
//
// Other splits that were measured on a 16 x 64 x 256 x 256 fp32 field with a gate per element, forward
// and backward: a thread per column of channels (no barriers, but two columns in registers leave 8
// warps per SM: 284 us and 2.1 ms); every thread adding all warps' parts itself (one barrier instead
// of two, but shared memory saturates: 452 and 558 us); 8-byte accesses, V = 2 and EPT = 4
// (296 and 526 us).  This one: 245 and 313 us, 0.96 of the measured HBM rate over both.
#pragma once

#include <algorithm>

#include "scx_internal.h"
#include "scx_residual_norm.cuh"

namespace scx_rn {
namespace {

constexpr int kMaxWarps = 16;
enum : int { kPostW = 0, kPostB = 1, kPreW = 2, kPreB = 3, kVectors = 4 };

template <int V, int EPT, int LC>
struct Shape {
    static constexpr int kPos = 32 / LC * V;         // positions of a tile
    static constexpr int kPerWarp = EPT * LC;        // channels of a warp
    static constexpr int kChannels = kMaxWarps * kPerWarp;
    static constexpr int kPitch = kPos + 8;          // float2 per row: neighbouring rows on other banks
    static constexpr int kPairs = EPT * V / 2;       // of a thread's values
    static constexpr int kSpots = V == 1 ? 1 : V / 2;  // pairs of a thread's positions
    static constexpr int kAcc = V == 1 ? EPT / 2 : EPT;
};

template <int V, int EPT, int LC>
struct alignas(16) Shared {
    using S = Shape<V, EPT, LC>;
    float vec[kVectors][S::kChannels];
    float2 part[kMaxWarps][S::kPitch];
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
    int warp, warps, pos, c0, mine, of_warp;  // mine, of_warp: channels that exist
    bool first;                               // of the warp's channel groups
};

template <int V, int EPT, int LC>
__device__ __forceinline__ Where where(const Problem& p) {
    constexpr int kLanes = 32 / LC;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int c0 = warp * EPT * LC + lane / kLanes * EPT;
    return {warp, static_cast<int>(blockDim.x) / 32, lane % kLanes, c0, max(0, min(EPT, p.channels - c0)),
            max(0, min(EPT * LC, p.channels - warp * EPT * LC)), lane < kLanes};
}

// A thread's values lie in pairs: two positions of one channel (V = 4: pairs 2j and 2j + 1 are channel
// j's), or two channels at one position (V = 1: pair i is channels 2i and 2i + 1).  Numbers per
// position come as pairs too, kSpots of them; for V = 1 the same number twice.
template <int V, int EPT>
struct Pairs {
    static constexpr int kCount = EPT * V / 2, kSpots = V == 1 ? 1 : V / 2;

    static __device__ __forceinline__ int spot(int i) { return V == 1 ? 0 : i % kSpots; }
    static __device__ __forceinline__ float2 channels(const float* of, int i) {
        return V == 1 ? make_float2(of[2 * i], of[2 * i + 1]) : both(of[i / kSpots]);
    }
    // sums over the thread's channels, per position
    static __device__ __forceinline__ void sum(const float2 (&v)[kCount], float2 (&s)[kSpots]) {
#pragma unroll
        for (int q = 0; q < kSpots; ++q) s[q] = v[q];
#pragma unroll
        for (int i = kSpots; i < kCount; ++i) s[spot(i)] = add2(s[spot(i)], v[i]);
        if (V == 1) s[0] = both(s[0].x + s[0].y);
    }
};

// Sums over the warp's channel groups.
template <int LC>
__device__ __forceinline__ float2 sum_groups(float2 v) {
#pragma unroll
    for (int o = 16; o >= 32 / LC && LC > 1; o >>= 1) {
        v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
        v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
    }
    return v;
}

// A few threads per position add the warps' parts: SHARES of them, each every SHARES-th warp.  WHOLE: the
// code of all steps at once, which is quicker by itself (training passes: 7x36x96x160 with a gate per sample
// 47 us against 49, 8x128x128x128 154 against 159).  With a gate per element in fp32, which HBM bounds, a loop
// (16x64x256x256: 559 us against 606; measured on that shape alone; what makes the difference is not known).
template <int SHARES, bool WHOLE>
struct Share {
    int me;

    // f over this share's warps
    template <typename F>
    __device__ __forceinline__ void for_warps(int warps, F f) const {
        if constexpr (WHOLE && SHARES > 1) {
#pragma unroll
            for (int k = 0; k < kMaxWarps / SHARES; ++k)
                if (k * SHARES + me < warps) f(k * SHARES + me);
        } else {
#pragma unroll 1
            for (int w = me; w < warps; w += SHARES) f(w);
        }
    }
    // the sum over the shares of a position, 8 lanes apart
    __device__ __forceinline__ float sum(float v) const {
#pragma unroll
        for (int o = 8; o < 8 * SHARES; o *= 2) v += __shfl_xor_sync(0xffffffffu, v, o);
        return v;
    }
};

// Joins two numbers per position and warp: f(share, position, whether it exists and is this thread's to
// store, read) runs on a few threads per position, read(w) being warp w's numbers, and its result comes
// back to every thread's positions in a and b.  Every thread of the block calls it.
template <bool WHOLE, int V, int EPT, int LC, typename F>
__device__ __forceinline__ void join(Shared<V, EPT, LC>& sh, const Where& at, float2 (&a)[Pairs<V, EPT>::kSpots],
                                     float2 (&b)[Pairs<V, EPT>::kSpots], F f) {
    using S = Shape<V, EPT, LC>;
    if (at.first) {
        float2* to = &sh.part[at.warp][at.pos * V];
        if constexpr (V == 1) {
            to[0] = make_float2(a[0].x, b[0].x);
        } else {
#pragma unroll
            for (int q = 0; q < S::kSpots; ++q)
                *reinterpret_cast<float4*>(to + 2 * q) = make_float4(a[q].x, b[q].x, a[q].y, b[q].y);
        }
    }
    __syncthreads();
    // whole warps take part or not: f shuffles
    const int lane = static_cast<int>(threadIdx.x % 32);
    auto one = [&](int q, auto share) {
        const bool here = q < S::kPos, store = here && share.me == 0;
        const float2* column = &sh.part[0][here ? q : 0];
        const float2 r = f(share, q, store, [&](int w) { return column[w * S::kPitch]; });
        if (store) sh.stat[q] = r;
    };
    if (S::kPos >= 8 && static_cast<int>(blockDim.x) >= 4 * S::kPos) {  // a warp: 8 positions x 4 shares
        if (at.warp < S::kPos / 8) one(at.warp * 8 + lane % 8, Share<4, WHOLE>{lane / 8});
    } else {
        for (int q0 = at.warp * 32; q0 < S::kPos; q0 += at.warps * 32) one(q0 + lane, Share<1, WHOLE>{0});
    }
    __syncthreads();
    const float2* from = &sh.stat[at.pos * V];
    if constexpr (V == 1) {
        a[0] = both(from[0].x);
        b[0] = both(from[0].y);
    } else {
#pragma unroll
        for (int s = 0; s < S::kSpots; ++s) {
            const float4 v = *reinterpret_cast<const float4*>(from + 2 * s);
            a[s] = make_float2(v.x, v.z);
            b[s] = make_float2(v.y, v.w);
        }
    }
}

// Rho = 1 / sqrt(variance + eps) and -mean rho over the channels of a thread's positions, so that the
// normalised value is v rho - mean rho; `keep` (may be null) receives mean and rho per position.
template <bool WHOLE, int V, int EPT, int LC>
__device__ __forceinline__ void statistics(Shared<V, EPT, LC>& sh, const Problem& p,
                                           const float2 (&v)[Pairs<V, EPT>::kCount], const Where& at,
                                           float2 (&rho)[Pairs<V, EPT>::kSpots], float2 (&shift)[Pairs<V, EPT>::kSpots],
                                           float* keep, int live_pos) {
    using P = Pairs<V, EPT>;
    constexpr int kPerWarp = EPT * LC;
    float2 d[P::kCount];
    const bool layer = p.kind == kLayer;
    if (layer) {  // channels that do not exist hold zeros
        P::sum(v, shift);
        const float2 inv = both(at.of_warp ? 1.f / static_cast<float>(at.of_warp) : 0.f);
#pragma unroll
        for (int q = 0; q < P::kSpots; ++q) shift[q] = mul2(sum_groups<LC>(shift[q]), inv);
#pragma unroll
        for (int i = 0; i < P::kCount; ++i) {
            const float2 m = shift[P::spot(i)];
            d[i] = add2(v[i], make_float2(-m.x, -m.y));
            if (V == 1) {
                if (2 * i >= at.mine) d[i].x = 0.f;
                if (2 * i + 1 >= at.mine) d[i].y = 0.f;
            } else if (i / P::kSpots >= at.mine) {
                d[i] = both(0.f);
            }
            d[i] = mul2(d[i], d[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < P::kCount; ++i) d[i] = mul2(v[i], v[i]);
#pragma unroll
        for (int q = 0; q < P::kSpots; ++q) shift[q] = both(0.f);
    }
    P::sum(d, rho);
#pragma unroll
    for (int q = 0; q < P::kSpots; ++q) rho[q] = sum_groups<LC>(rho[q]);
    join<WHOLE, V, EPT, LC>(sh, at, shift, rho, [&](auto share, int q, bool store, auto part) {
        float mean = 0.f, sum = 0.f;
        if (layer) {
            auto count = [&](int w) { return static_cast<float>(min(kPerWarp, p.channels - w * kPerWarp)); };
            share.for_warps(at.warps, [&](int w) { mean = fmaf(count(w), part(w).x, mean); });
            mean = share.sum(mean) * p.inv_c;
            share.for_warps(at.warps, [&](int w) {
                const float2 e = part(w);
                const float off = e.x - mean;
                sum += fmaf(count(w) * off, off, e.y);
            });
        } else {
            share.for_warps(at.warps, [&](int w) { sum += part(w).y; });
        }
        const float r = rsqrtf(fmaf(share.sum(sum), p.inv_c, p.eps));
        if (store && keep != nullptr && q < live_pos) {
            keep[q] = mean;
            keep[p.positions + q] = r;
        }
        return make_float2(-mean * r, r);
    });
}

// The negatives of the means over the channels of two products, given as sums over the thread's
// channels per position; the first is zero in the RMS kind.
template <bool WHOLE, int V, int EPT, int LC>
__device__ __forceinline__ void two_means(Shared<V, EPT, LC>& sh, const Problem& p, const Where& at,
                                          float2 (&m1)[Pairs<V, EPT>::kSpots], float2 (&m2)[Pairs<V, EPT>::kSpots]) {
    const bool layer = p.kind == kLayer;
#pragma unroll
    for (int q = 0; q < Pairs<V, EPT>::kSpots; ++q) {
        if (layer) m1[q] = sum_groups<LC>(m1[q]);
        m2[q] = sum_groups<LC>(m2[q]);
    }
    join<WHOLE, V, EPT, LC>(sh, at, m1, m2, [&](auto share, int, bool, auto part) {
        float2 s = both(0.f);
        share.for_warps(at.warps, [&](int w) { s = add2(s, part(w)); });
        return make_float2(layer ? -share.sum(s.x) * p.inv_c : 0.f, -share.sum(s.y) * p.inv_c);
    });
}

template <typename T, int MODE>
constexpr bool kWhole = sizeof(T) == 2 || MODE != kFull;

// Where a tile lies, for one thread; moved on by `step` tiles without a division.
template <int V, int EPT, int LC>
struct Tile {
    int sample, index;  // the tile's index in its sample

    __device__ __forceinline__ Tile(const Problem& p, int tile) {
        const int per_sample = static_cast<int>(p.tiles_per_sample);
        sample = tile / per_sample;
        index = tile - sample * per_sample;
    }
    __device__ __forceinline__ void next(const Problem& p, int step_samples, int step_index) {
        sample += step_samples;
        index += step_index;
        if (index >= static_cast<int>(p.tiles_per_sample)) {
            index -= static_cast<int>(p.tiles_per_sample);
            ++sample;
        }
    }
    __device__ __forceinline__ int l0() const { return index * Shape<V, EPT, LC>::kPos; }
    // whether the thread's positions exist, and its first element
    __device__ __forceinline__ bool live(const Problem& p, const Where& at) const {
        return l0() + at.pos * V < static_cast<int>(p.length);
    }
    __device__ __forceinline__ size_t base(const Problem& p, const Where& at) const {
        return (static_cast<size_t>(sample) * p.channels + at.c0) * p.length + (l0() + at.pos * V);
    }
};

// Where a thread's channels of one tile lie in a tensor, in bytes; the tensor's start where there is
// nothing.
template <int EPT>
struct Spots {
    size_t at[EPT];
    bool live[EPT];
};

// A thread's slots in shared memory, and how it fills and reads them: slot k is a tensor of a tile, EPT
// vectors, `pitch` bytes apart.
template <typename T, int V, int EPT>
struct Slots {
    using E = Vec<T, V>;
    using P = Pairs<V, EPT>;
    unsigned char* base;
    unsigned address, pitch;
    size_t stride;  // from channel to channel, in bytes
    int mine;

    __device__ __forceinline__ Slots(unsigned char* shared, const Problem& p, const Where& at)
        : base(shared + threadIdx.x * sizeof(E)), address(shared_address(base)), pitch(blockDim.x * sizeof(E)),
          stride(static_cast<size_t>(p.length) * sizeof(T)), mine(at.mine) {}

    // `first`: the thread's first element
    __device__ __forceinline__ Spots<EPT> spots(size_t first, bool live) const {
        Spots<EPT> s;
        const size_t bytes = live && mine > 0 ? first * sizeof(T) : 0;
#pragma unroll
        for (int j = 0; j < EPT; ++j) {
            s.live[j] = live && j < mine;
            s.at[j] = bytes + (j < mine && live ? j * stride : 0);
        }
        return s;
    }

    __device__ __forceinline__ void fetch(unsigned k, const void* from, const Spots<EPT>& s) const {
        if constexpr (kCopied<E>) {
#pragma unroll
            for (int j = 0; j < EPT; ++j)
                copy_async<E>(address + (k * EPT + j) * pitch, static_cast<const char*>(from) + s.at[j], s.live[j]);
        }
    }

    __device__ __forceinline__ void read(unsigned k, const void* from, const Spots<EPT>& s, float2 (&out)[P::kCount]) const {
        E v[EPT];
#pragma unroll
        for (int j = 0; j < EPT; ++j) {
            v[j] = E{};
            if constexpr (kCopied<E>) v[j] = *reinterpret_cast<const E*>(base + (k * EPT + j) * pitch);
            else if (s.live[j]) v[j] = *reinterpret_cast<const E*>(static_cast<const char*>(from) + s.at[j]);
        }
#pragma unroll
        for (int i = 0; i < P::kCount; ++i) {
            if constexpr (V == 1) out[i] = make_float2(v[2 * i].one(), v[2 * i + 1].one());
            else out[i] = v[i / P::kSpots].pair(i % P::kSpots);
        }
    }

    __device__ __forceinline__ void store(void* to, const Spots<EPT>& s, const float2 (&v)[P::kCount]) const {
        E o[EPT];
#pragma unroll
        for (int i = 0; i < P::kCount; ++i) {
            if constexpr (V == 1) {
                o[2 * i].set_one(v[i].x);
                o[2 * i + 1].set_one(v[i].y);
            } else {
                o[i / P::kSpots].set_pair(i % P::kSpots, v[i]);
            }
        }
#pragma unroll
        for (int j = 0; j < EPT; ++j)
            if (s.live[j]) *reinterpret_cast<E*>(static_cast<char*>(to) + s.at[j]) = o[j];
    }
};

// act(gate) of a thread's channels, the gate being one value per sample and channel.
template <typename T, int V, int EPT>
__device__ __forceinline__ void sample_gate(const Problem& p, const Where& at, int sample,
                                            float2 (&a)[Pairs<V, EPT>::kCount]) {
    float g[EPT];
#pragma unroll
    for (int j = 0; j < EPT; ++j)
        g[j] = j < at.mine ? activate(to_f32(static_cast<const T*>(
                                          p.gate)[static_cast<size_t>(sample) * p.channels + at.c0 + j]), p.act)
                           : 0.f;
#pragma unroll
    for (int i = 0; i < Pairs<V, EPT>::kCount; ++i) a[i] = Pairs<V, EPT>::channels(g, i);
}

__host__ __device__ constexpr int forward_tensors(int mode) { return mode == kNoBlock ? 1 : mode == kFull ? 3 : 2; }

template <typename T, int V, int EPT, int LC, int MODE>
__global__ void __launch_bounds__(kMaxWarps * 32, 2) field_forward_kernel(const __grid_constant__ Problem p) {
    using F = Slots<T, V, EPT>;
    using P = Pairs<V, EPT>;
    extern __shared__ __align__(16) unsigned char dynamic[];
    auto& sh = *reinterpret_cast<Shared<V, EPT, LC>*>(dynamic);
    const Where at = where<V, EPT, LC>(p);
    const int tiles = static_cast<int>(p.tiles);
    constexpr int kTensors = forward_tensors(MODE);
    const F slots(dynamic + sizeof(sh), p, at);
    using TILE = Tile<V, EPT, LC>;
    auto fetch = [&](const TILE& t, bool exists, int turn) {
        if (exists) {
            const Spots<EPT> spots = slots.spots(t.base(p, at), t.live(p, at));
            const unsigned k = turn * kTensors;
            slots.fetch(k, p.x, spots);
            if constexpr (MODE != kNoBlock) slots.fetch(k + 1, p.y, spots);
            if constexpr (MODE == kFull) slots.fetch(k + 2, p.gate, spots);
        }
        copy_commit();
    };
    TILE t(p, blockIdx.x);
    const TILE step(p, gridDim.x);  // as a number of samples and of tiles
    fetch(t, static_cast<int>(blockIdx.x) < tiles, 0);
    load_vectors<T>(sh, p, at.warps * EPT * LC);
    int turn = 0;
    for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x, turn ^= 1) {
        const Spots<EPT> spots = slots.spots(t.base(p, at), t.live(p, at));
        const int sample = t.sample;
        const unsigned slot = turn * kTensors;
        const size_t q0 = static_cast<size_t>(sample) * p.length + t.l0();
        const int live_pos = static_cast<int>(p.length) - t.l0();
        t.next(p, step.sample, step.index);
        fetch(t, tile + static_cast<int>(gridDim.x) < tiles, turn ^ 1);
        copy_wait<1>();
        float2 r[P::kCount], rho[P::kSpots], shift[P::kSpots];
        slots.read(slot, p.x, spots, r);
        if constexpr (MODE != kNoBlock) {
            float2 h[P::kCount], a[P::kCount];
            slots.read(slot + 1, p.y, spots, h);
            if constexpr (MODE == kFull) slots.read(slot + 2, p.gate, spots, a);
            if (p.post) {
                statistics<kWhole<T, MODE>, V, EPT, LC>(sh, p, h, at, rho, shift, p.stats ? p.stats + q0 : nullptr, live_pos);
#pragma unroll
                for (int i = 0; i < P::kCount; ++i) h[i] = fma2(h[i], rho[P::spot(i)], shift[P::spot(i)]);
            }
            if constexpr (MODE == kFull) activate_all<T>(a, p.act);
            if constexpr (MODE == kSample) sample_gate<T, V, EPT>(p, at, sample, a);
#pragma unroll
            for (int i = 0; i < P::kCount; ++i) {
                const float2 z = fma2(h[i], P::channels(&sh.vec[kPostW][at.c0], i), P::channels(&sh.vec[kPostB][at.c0], i));
                r[i] = MODE == kPlain ? add2(r[i], z) : fma2(a[i], z, r[i]);
            }
            slots.store(p.r, spots, r);
        }
        if (!p.pre) continue;
        statistics<kWhole<T, MODE>, V, EPT, LC>(sh, p, r, at, rho, shift, p.stats ? p.stats + 2 * p.positions + q0 : nullptr, live_pos);
#pragma unroll
        for (int i = 0; i < P::kCount; ++i)
            r[i] = fma2(fma2(r[i], rho[P::spot(i)], shift[P::spot(i)]), P::channels(&sh.vec[kPreW][at.c0], i),
                        P::channels(&sh.vec[kPreB][at.c0], i));
        slots.store(p.n, spots, r);
    }
    copy_wait<0>();
}

// The forward's statistics of a thread's positions; zero rho where there is no position.  They are
// loaded a tile ahead, like the tensors.
template <int V>
struct Saved {
    static constexpr int kSpots = V == 1 ? 1 : V / 2;
    float2 mean[kSpots], rho[kSpots], mean2[kSpots], rho2[kSpots];

    template <typename TILE>
    __device__ __forceinline__ void load(const Problem& p, const TILE& t, const Where& at) {
#pragma unroll
        for (int s = 0; s < kSpots; ++s) mean[s] = rho[s] = mean2[s] = rho2[s] = both(0.f);
        if (!t.live(p, at)) return;
        // V divides the length, so V positions' numbers of one kind are one aligned access
        const size_t q = static_cast<size_t>(t.sample) * p.length + t.l0() + at.pos * V, row = static_cast<size_t>(p.positions);
        auto read = [&](size_t from, float2 (&to)[kSpots]) {
            const float* v = p.stats + from;
#pragma unroll
            for (int s = 0; s < kSpots; ++s) to[s] = V == 1 ? both(v[0]) : make_float2(v[2 * s % V], v[(2 * s + 1) % V]);
        };
#pragma unroll
        for (int s = 0; s < kSpots; ++s) rho[s] = both(1.f);
        if (p.post) {
            read(q, mean);
            read(row + q, rho);
        }
        if (p.dn) {
            read(2 * row + q, mean2);
            read(3 * row + q, rho2);
        }
    }
};

// Adds v over the lanes that share this lane's channel group.
template <int LC>
__device__ __forceinline__ float sum_positions(float v) {
#pragma unroll
    for (int o = 16 / LC; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Tensors a backward reads: x, y, dn, dr, and a gate per element.
__host__ __device__ constexpr int backward_tensors(int mode) { return mode == kFull ? 5 : 4; }

// MAXW: the most warps it is launched with.  Up to 10 the registers are held to what lets two blocks
// share an SM (36 channels of 7 x 96 x 160 with a gate per sample: 30 us against 40 us).  With a gate per element
// that spills 52 to 56 bytes of the 10 warps' kernel, as the forward's two blocks per SM do up to 80 of the kernels
// by single values.
template <typename T, int V, int EPT, int LC, int MODE, int MAXW>
__global__ void __launch_bounds__(MAXW * 32, MAXW <= 10 ? 2 : 1) field_backward_kernel(const __grid_constant__ Problem p) {
    using F = Slots<T, V, EPT>;
    using P = Pairs<V, EPT>;
    using TILE = Tile<V, EPT, LC>;
    constexpr int N = P::kCount, kSpots = P::kSpots, kAcc = Shape<V, EPT, LC>::kAcc;
    extern __shared__ __align__(16) unsigned char dynamic[];
    auto& sh = *reinterpret_cast<Shared<V, EPT, LC>*>(dynamic);
    grid_dep_launch();
    const Where at = where<V, EPT, LC>(p);
    constexpr int kTensors = backward_tensors(MODE);
    const F slots(dynamic + sizeof(sh), p, at);
    // Tiles in a row across the blocks, so that what is under way at one time lies together in DRAM's pages
    // (a training pass of 16x64x129x129 in fp32: 308 us, with a run of tiles per block 330).  With a gate per
    // sample a run of tiles per block all the same: its sums are kept by sample.
    const int first = MODE == kSample ? static_cast<int>(tile_begin(p, blockIdx.x)) : blockIdx.x;
    const int last = static_cast<int>(MODE == kSample ? tile_begin(p, blockIdx.x + 1) : p.tiles);
    const int stride = MODE == kSample ? 1 : gridDim.x;
    Saved<V> ahead;
    auto fetch = [&](const TILE& t, bool exists, int turn) {
        if (exists) {
            const Spots<EPT> spots = slots.spots(t.base(p, at), t.live(p, at));
            const unsigned k = turn * kTensors;
            if constexpr (MODE != kNoBlock) slots.fetch(k + 1, p.y, spots);
            if (p.dn) {
                slots.fetch(k, p.x, spots);
                slots.fetch(k + 2, p.dn, spots);
            }
            if (p.dr) slots.fetch(k + 3, p.dr, spots);
            if constexpr (MODE == kFull) slots.fetch(k + 4, p.gate, spots);
            ahead.load(p, t, at);
        }
        copy_commit();
    };
    TILE t(p, first);
    const TILE step(p, stride);
    fetch(t, first < last, 0);
    load_vectors<T>(sh, p, at.warps * EPT * LC);
    int turn = 0;
    // sums over positions: per channel (V = 4: to be added over the pair), or per pair of channels
    float2 sum[kSums][kAcc];
#pragma unroll
    for (int k = 0; k < kSums; ++k)
#pragma unroll
        for (int i = 0; i < kAcc; ++i) sum[k][i] = both(0.f);
    auto acc = [](int i) { return V == 1 ? i : i / kSpots; };
    auto of_channel = [&](int kind, int j) {
        return V == 1 ? (j % 2 ? sum[kind][j / 2].y : sum[kind][j / 2].x) : sum[kind][j % kAcc].x + sum[kind][j % kAcc].y;
    };
    for (int tile = first; tile < last; tile += stride, turn ^= 1) {
        const Spots<EPT> spots = slots.spots(t.base(p, at), t.live(p, at));
        const int sample = t.sample;
        const unsigned slot = turn * kTensors;
        const bool sample_ends = t.index + 1 == static_cast<int>(p.tiles_per_sample);
        float2 rho[kSpots], shift[kSpots], rho2[kSpots], shift2[kSpots];
#pragma unroll
        for (int s = 0; s < kSpots; ++s) {
            rho[s] = ahead.rho[s];
            rho2[s] = ahead.rho2[s];
            shift[s] = make_float2(-ahead.mean[s].x * rho[s].x, -ahead.mean[s].y * rho[s].y);
            shift2[s] = make_float2(-ahead.mean2[s].x * rho2[s].x, -ahead.mean2[s].y * rho2[s].y);
        }
        t.next(p, MODE == kSample ? 0 : step.sample, MODE == kSample ? 1 : step.index);
        fetch(t, tile + stride < last, turn ^ 1);
        copy_wait<1>();
        float2 h[N], a[N], slope[N], k[N], g[N];
        if constexpr (MODE != kNoBlock) {
            slots.read(slot + 1, p.y, spots, h);
#pragma unroll
            for (int i = 0; i < N; ++i) h[i] = fma2(h[i], rho[P::spot(i)], shift[P::spot(i)]);
            if constexpr (MODE == kFull) {
                slots.read(slot + 4, p.gate, spots, a);
                activate_all<T>(a, slope, p.act);
            }
            if constexpr (MODE == kSample) sample_gate<T, V, EPT>(p, at, sample, a);
        }
        if (p.dn) {
            slots.read(slot + 0, p.x, spots, k);
            slots.read(slot + 2, p.dn, spots, g);
            float2 gk[N], m1[kSpots], m2[kSpots];
#pragma unroll
            for (int i = 0; i < N; ++i) {
                if constexpr (MODE != kNoBlock) {
                    const float2 z =
                        fma2(h[i], P::channels(&sh.vec[kPostW][at.c0], i), P::channels(&sh.vec[kPostB][at.c0], i));
                    k[i] = MODE == kPlain ? add2(k[i], z) : fma2(a[i], z, k[i]);
                }
                k[i] = fma2(k[i], rho2[P::spot(i)], shift2[P::spot(i)]);
                sum[kDPreW][acc(i)] = fma2(g[i], k[i], sum[kDPreW][acc(i)]);
                sum[kDPreB][acc(i)] = add2(sum[kDPreB][acc(i)], g[i]);
                g[i] = mul2(g[i], P::channels(&sh.vec[kPreW][at.c0], i));
                gk[i] = mul2(g[i], k[i]);
            }
            P::sum(g, m1);
            P::sum(gk, m2);
            two_means<kWhole<T, MODE>, V, EPT, LC>(sh, p, at, m1, m2);
#pragma unroll
            for (int i = 0; i < N; ++i)
                g[i] = mul2(rho2[P::spot(i)], add2(fma2(k[i], m2[P::spot(i)], g[i]), m1[P::spot(i)]));
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) g[i] = both(0.f);
        }
        if (p.dr) {
            slots.read(slot + 3, p.dr, spots, k);
#pragma unroll
            for (int i = 0; i < N; ++i) g[i] = add2(g[i], k[i]);
        }
        // g: the gradient of r
        if (p.dx) slots.store(p.dx, spots, g);
        if constexpr (MODE != kNoBlock) {
            float2 kh[N];
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float2 ta = MODE == kPlain ? g[i] : mul2(g[i], a[i]);
                const float2 v = MODE == kSample ? g[i] : ta;
                sum[kTah][acc(i)] = fma2(v, h[i], sum[kTah][acc(i)]);
                sum[kTa][acc(i)] = add2(sum[kTa][acc(i)], v);
                k[i] = mul2(ta, P::channels(&sh.vec[kPostW][at.c0], i));
                kh[i] = mul2(k[i], h[i]);
            }
            if (MODE == kFull && p.dgate) {
#pragma unroll
                for (int i = 0; i < N; ++i)
                    a[i] = mul2(mul2(g[i], slope[i]),
                                fma2(h[i], P::channels(&sh.vec[kPostW][at.c0], i), P::channels(&sh.vec[kPostB][at.c0], i)));
                slots.store(p.dgate, spots, a);
            }
            if (p.dy) {
                if (p.post) {
                    float2 m1[kSpots], m2[kSpots];
                    P::sum(k, m1);
                    P::sum(kh, m2);
                    two_means<kWhole<T, MODE>, V, EPT, LC>(sh, p, at, m1, m2);
#pragma unroll
                    for (int i = 0; i < N; ++i)
                        k[i] = mul2(rho[P::spot(i)], add2(fma2(h[i], m2[P::spot(i)], k[i]), m1[P::spot(i)]));
                }
                slots.store(p.dy, spots, k);
            }
            if (MODE == kSample && p.slots && (tile + 1 == last || sample_ends)) {
                float* to = slot_of(p, blockIdx.x, sample);
#pragma unroll
                for (int j = 0; j < EPT; ++j) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float total = sum_positions<LC>(of_channel(kTah + i, j));
                        if (at.pos == 0 && j < at.mine) to[static_cast<size_t>(i) * p.channels + at.c0 + j] = total;
                    }
                }
#pragma unroll
                for (int i = 0; i < kAcc; ++i) sum[kTah][i] = sum[kTa][i] = both(0.f);
            }
        }
    }
    copy_wait<0>();
    if (!p.sums) return;
#pragma unroll
    for (int i = 0; i < kSums; ++i) {
#pragma unroll
        for (int j = 0; j < EPT; ++j) {
            const float total = sum_positions<LC>(of_channel(i, j));
            if (at.pos == 0 && j < at.mine)
                p.partial[(static_cast<size_t>(blockIdx.x) * kSums + i) * p.channels + at.c0 + j] = total;
        }
    }
}

// Sets the tiles of a shape; false where their count or a position does not fit the kernels' int.
template <typename S>
bool set_tiles(Problem& p) {
    p.tiles_per_sample = (p.length + S::kPos - 1) / S::kPos;
    p.tiles = p.batch * p.tiles_per_sample;
    return p.tiles < (1LL << 30) && p.length < (1LL << 30);
}

template <typename S>
int threads_for(int channels) {
    return (channels + S::kPerWarp - 1) / S::kPerWarp * 32;
}

template <typename T, int V, int EPT, int LC, int MODE>
cudaError_t forward_as(Problem p, cudaStream_t s) {
    using S = Shape<V, EPT, LC>;
    if (!set_tiles<S>(p)) return cudaErrorNotSupported;
    const int threads = threads_for<S>(p.channels);
    const size_t smem = sizeof(Shared<V, EPT, LC>) +
                        (kCopied<Vec<T, V>> ? 2 * forward_tensors(MODE) * EPT * sizeof(Vec<T, V>) * threads : 0);
    int per_sm = 0;
    const cudaError_t e = scx::prepare_kernel(reinterpret_cast<const void*>(field_forward_kernel<T, V, EPT, LC, MODE>),
                                              smem, threads, &per_sm);
    if (e != cudaSuccess) return e;
    const int grid = static_cast<int>(std::min<long long>(p.tiles, static_cast<long long>(per_sm) * scx::num_sms()));
    field_forward_kernel<T, V, EPT, LC, MODE><<<grid, threads, smem, s>>>(p);
    return cudaGetLastError();
}

template <typename T, int V, int EPT, int LC, int MODE, int MAXW = kMaxWarps>
cudaError_t backward_as(Problem& p, cudaStream_t s) {
    using S = Shape<V, EPT, LC>;
    Problem q = p;
    if (!set_tiles<S>(q)) return cudaErrorNotSupported;
    const int threads = threads_for<S>(p.channels);
    const size_t smem = sizeof(Shared<V, EPT, LC>) +
                        (kCopied<Vec<T, V>> ? 2 * backward_tensors(MODE) * EPT * sizeof(Vec<T, V>) * threads : 0);
    int per_sm = 0;
    const cudaError_t e = scx::prepare_kernel(reinterpret_cast<const void*>(field_backward_kernel<T, V, EPT, LC, MODE, MAXW>),
                                              smem, threads, &per_sm);
    if (e != cudaSuccess) return e;
    q.parts = static_cast<int>(std::min<long long>(std::min(max_parts(p.channels), per_sm * scx::num_sms()), q.tiles));
    q.partials = q.parts;
    p = q;
    field_backward_kernel<T, V, EPT, LC, MODE, MAXW><<<p.parts, threads, smem, s>>>(p);
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

// The more channels, the fewer positions a tile has: as many as 16 warps of 8 values per thread leave.  Two-byte
// fields of more than 256 channels, whose vectors of 4 would be half a sector or less, go by single positions
// and more channels per thread (2x768x128x128 bf16 training pass 664 us, by vectors 871; 512 channels 600 and
// 653; 256 channels 507 and 462).
template <typename T, int MODE>
cudaError_t forward_in(const Problem& p, cudaStream_t s) {
    if (vectors_fit<T, 4>(p)) {
        if (p.channels <= 64) return forward_as<T, 4, 2, 2, MODE>(p, s);
        if (p.channels <= 128) return forward_as<T, 4, 2, 4, MODE>(p, s);
        if (p.channels <= 256) return forward_as<T, 4, 2, 8, MODE>(p, s);
        if constexpr (sizeof(T) == 4) {
            if (p.channels <= 512) return forward_as<T, 4, 2, 16, MODE>(p, s);
            if (p.channels <= 1024) return forward_as<T, 4, 2, 32, MODE>(p, s);
        }
    }
    if (p.channels <= 128) return forward_as<T, 1, 8, 1, MODE>(p, s);
    if (p.channels <= 256) return forward_as<T, 1, 8, 2, MODE>(p, s);
    if (p.channels <= 512) return forward_as<T, 1, 8, 4, MODE>(p, s);
    if (p.channels <= 1024) return forward_as<T, 1, 8, 8, MODE>(p, s);
    return cudaErrorNotSupported;
}

template <typename T, int MODE>
cudaError_t backward_in(Problem& p, cudaStream_t s) {
    if (vectors_fit<T, 4>(p)) {
        if (p.channels <= 32) return backward_as<T, 4, 2, 2, MODE, 8>(p, s);
        if (p.channels <= 40) return backward_as<T, 4, 2, 2, MODE, 10>(p, s);
        if (p.channels <= 64) return backward_as<T, 4, 2, 2, MODE>(p, s);
        if (p.channels <= 128) return backward_as<T, 4, 2, 4, MODE>(p, s);
        if (p.channels <= 256) return backward_as<T, 4, 2, 8, MODE>(p, s);
        if constexpr (sizeof(T) == 4) {
            if (p.channels <= 512) return backward_as<T, 4, 2, 16, MODE>(p, s);
            if (p.channels <= 1024) return backward_as<T, 4, 2, 32, MODE>(p, s);
        }
    }
    if (p.channels <= 64) return backward_as<T, 1, 8, 1, MODE, 8>(p, s);
    if (p.channels <= 128) return backward_as<T, 1, 8, 1, MODE>(p, s);
    if (p.channels <= 256) return backward_as<T, 1, 8, 2, MODE>(p, s);
    if (p.channels <= 512) return backward_as<T, 1, 8, 4, MODE>(p, s);
    if (p.channels <= 1024) return backward_as<T, 1, 8, 8, MODE>(p, s);
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
