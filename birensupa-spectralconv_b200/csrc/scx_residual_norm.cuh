// What the residual-norm kernels share: a call's description, loads and stores by type, the gate's
// activation, and how a backward's blocks split the positions.
#pragma once

#include <cstdint>

#include <cuda_runtime.h>

#include "scx_vec.cuh"

namespace scx_rn {

using scx::from_f32;
using scx::load_vec;
using scx::store_vec;
using scx::to_f32;
using scx::Vec;

enum : int { kF32 = 0, kBf16 = 1, kF16 = 2 };
enum : int { kRms = 0, kLayer = 1 };
enum : int { kGateNone = 0, kGateSample = 1, kGateFull = 2 };
enum : int { kActNone = 0, kActSigmoid = 1, kActSilu = 2 };

// A call's shapes, options and addresses, as a kernel parameter.
struct Problem {
    long long batch, length, positions;  // positions = batch * length
    int channels;
    int channels_last;
    int kind, gate_mode, act;
    int post, pre;  // whether the norm after the block, and the one before the next, is taken
    int wide;       // weights are fp32 rather than the tensors' type
    float eps, inv_c, scale;
    const void *x, *y, *gate, *post_w, *post_b, *pre_w, *pre_b, *scale_w;
    void *r, *n;
    float* stats;  // post mean, post rho, pre mean, pre rho: [positions][4] of tokens, [4][positions] of fields
    const void *dr, *dn;
    void *dx, *dy, *dgate, *d_post_w, *d_post_b, *d_pre_w, *d_pre_b, *d_scale;
    int sums;        // whether any gradient summed over positions is wanted
    float* means;    // [2][positions]: mean(dn w'), mean(dn w' k); any-shape kernels only
    float* partial;  // [partials][kSums][channels]
    float* slots;    // [parts + batch][2][channels], with a gate per sample whose sums are wanted
    long long tiles, tiles_per_sample;  // a tile: some positions of one sample
    int parts;                          // blocks or warps that share the tiles
    int partials;                       // rows of `partial`
};

// The sums over positions that a backward's blocks leave per channel.  With a = act(gate):
//   dw' = sum dn k, db' = sum dn, and from A = sum t a h, B = sum t a:
//   dw = scale A, db = scale B, dscale = w A + b B (z = w h + b), dgate of a sample, whose a is
//   constant, from sum t h and sum t over its positions.
// With a gate per sample the last two are kept per sample, without a, in `slots`.
enum : int { kDPreW = 0, kDPreB = 1, kTah = 2, kTa = 3, kSums = 4 };

// Part b of a backward (a block, or a warp) takes the tiles [tile_begin(b), tile_begin(b + 1)), in order.
__host__ __device__ __forceinline__ long long tile_begin(const Problem& p, long long b) {
    return p.tiles * b / p.parts;
}

// The part that has tile t: the largest b with tile_begin(b) <= t.
__host__ __device__ __forceinline__ long long part_of_tile(const Problem& p, long long t) {
    return ((t + 1) * p.parts - 1) / p.tiles;
}

// Where part b keeps its sums over its positions of sample s: b + s grows by one with either, so
// no two (part, sample) pairs that meet share a slot.
__device__ __forceinline__ float* slot_of(const Problem& p, long long b, long long s) {
    return p.slots + static_cast<size_t>(b + s) * 2 * p.channels;
}

__device__ __forceinline__ void grid_dep_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_dep_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// Two fp32 values at once: sm_100a has packed fp32 arithmetic, which halves the instructions of
// these kernels' inner loops (the token kernels in bf16 are bound by them).
__device__ __forceinline__ float2 both(float a) { return make_float2(a, a); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 add2(float2 a, float2 b) { return __fadd2_rn(a, b); }

template <typename T>
__device__ __forceinline__ float weight(const void* w, int c, bool wide, float other) {
    if (w == nullptr) return other;
    return wide ? static_cast<const float*>(w)[c] : to_f32(static_cast<const T*>(w)[c]);
}

template <typename T>
__device__ __forceinline__ void store_weight(void* w, int c, bool wide, float v) {
    if (wide) static_cast<float*>(w)[c] = v;
    else from_f32(static_cast<T*>(w)[c], v);
}

// Reciprocal and power of two from the hardware's approximations (PTX rcp and ex2, both within a few
// units in the last place), and bounds that keep NaN.
__device__ __forceinline__ float rcp_approx(float v) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float exp2_approx(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float within(float v, float bound) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(v), "f"(bound));
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(r), "f"(-bound));
    return r;
}

// 1 / (1 + exp(-g)) of a pair.  exp(-g) = 2^t (1 + ln2 (t* - t)) with t* = -g log2(e) and t its rounding:
// the difference comes exactly from a fused product, with log2(e) in two parts, so that the error
// does not grow with g.  Relative error below 8 roundings down to g = -87, where the result leaves
// the normal numbers and is zero.  For gates of two bytes 2^t alone: the rounding of t costs |g| 2^-24, at
// most 2^-17.5, a ninetieth of fp16's own (8192x2048 bf16 tokens 107.3 us, with the correction 110.6).  The fp32 sums
// over positions take it in too: as an absolute error that is 1.25 |g| s (1 - s) 2^-24, below a third of a
// rounding of one.
template <typename T>
__device__ __forceinline__ float2 sigmoid2(float2 g) {
    constexpr float kLog2e = 1.44269504f, kLog2eRest = 1.92596299e-8f, kLn2 = 0.69314718f;
    if constexpr (sizeof(T) == 4) g = make_float2(within(g.x, 88.f), within(g.y, 88.f));  // 2^t stays finite
    const float2 t = mul2(g, both(-kLog2e));
    float2 e = make_float2(exp2_approx(t.x), exp2_approx(t.y));
    if constexpr (sizeof(T) == 4) {
        const float2 over = fma2(g, both(kLog2eRest), fma2(g, both(kLog2e), t));  // t - t*
        e = fma2(mul2(e, both(-kLn2)), over, e);
    }
    e = add2(e, both(1.f));
    return make_float2(rcp_approx(e.x), rcp_approx(e.y));
}
__device__ __forceinline__ float sigmoid(float g) { return sigmoid2<float>(both(g)).x; }

// act(g) and its derivative.
__device__ __forceinline__ float activate(float g, int act, float& slope) {
    if (act == kActNone) {
        slope = 1.f;
        return g;
    }
    const float s = sigmoid(g);
    if (act == kActSilu) {
        slope = s * (1.f + g * (1.f - s));
        return g * s;
    }
    slope = s * (1.f - s);
    return s;
}

__device__ __forceinline__ float activate(float g, int act) {
    float slope;
    return activate(g, act, slope);
}

// act over a thread's pairs, the choice made once; one copy of the sigmoid keeps the loop's code short.
template <typename T, int P>
__device__ __forceinline__ void activate_all(float2 (&g)[P], int act) {
    if (act == kActNone) return;
    float2 s[P];
#pragma unroll
    for (int i = 0; i < P; ++i) s[i] = sigmoid2<T>(g[i]);
#pragma unroll
    for (int i = 0; i < P; ++i) g[i] = act == kActSilu ? mul2(g[i], s[i]) : s[i];
}

// The same and the derivative.
template <typename T, int P>
__device__ __forceinline__ void activate_all(float2 (&g)[P], float2 (&slope)[P], int act) {
#pragma unroll
    for (int i = 0; i < P; ++i) slope[i] = both(1.f);
    if (act == kActNone) return;
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const float2 s = sigmoid2<T>(g[i]), rest = make_float2(1.f - s.x, 1.f - s.y);
        if (act == kActSilu) {
            g[i] = mul2(g[i], s);
            slope[i] = fma2(g[i], rest, s);
        } else {
            g[i] = s;
            slope[i] = mul2(s, rest);
        }
    }
}

// What a kernel's code depends on: whether there is a block's output, and a gate of which form.
enum Mode : int { kNoBlock = 0, kPlain = 1, kSample = 2, kFull = 3 };

inline int mode_of(const Problem& p) {
    return p.y == nullptr ? kNoBlock : p.gate_mode == kGateNone ? kPlain : p.gate_mode == kGateSample ? kSample : kFull;
}

// A thread's copies from global to its own slots in shared memory, ahead of their use: they need no
// registers while in flight, and no barrier, since nobody else reads the slots.  `live` false
// fills with zeros.  Copies are of 4, 8 or 16 bytes; narrower vectors (kCopied false) are loaded
// when they are used.
template <typename V>
constexpr bool kCopied = sizeof(V) >= 4;

__device__ __forceinline__ unsigned shared_address(const void* p) {
    return static_cast<unsigned>(__cvta_generic_to_shared(p));
}

template <typename V>
__device__ __forceinline__ void copy_async(unsigned dst, const void* from, bool live) {
    const int bytes = live ? static_cast<int>(sizeof(V)) : 0;
    if constexpr (sizeof(V) == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(from), "r"(bytes) : "memory");
    else if constexpr (sizeof(V) == 8)
        asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(from), "r"(bytes) : "memory");
    else if constexpr (sizeof(V) == 4)
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(from), "r"(bytes) : "memory");
}

__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }

template <int N>
__device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Launchers of the kernels that keep a position's channels in registers.  They return
// cudaErrorNotSupported, without a launch, for a problem they do not take.  The backward ones set
// p.tiles, p.tiles_per_sample and p.parts for the sums that follow.
template <typename T>
cudaError_t field_forward(const Problem& p, cudaStream_t s);
template <typename T>
cudaError_t field_backward(Problem& p, cudaStream_t s);
template <typename T>
cudaError_t token_forward(const Problem& p, cudaStream_t s);
template <typename T>
cudaError_t token_backward(Problem& p, cudaStream_t s);

// Most parts that share a backward's tiles; bounds `partial` to 64 MB at any channel count.
inline int max_parts(int channels) {
    const int n = (1 << 22) / channels;
    return n < 16 ? 16 : n > 4096 ? 4096 : n;
}

inline bool aligned(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

}  // namespace scx_rn
