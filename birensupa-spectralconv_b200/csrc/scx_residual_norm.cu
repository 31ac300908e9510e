// The norms after and before a block, fused with the block's gate, residual scale and residual
// addition, forward and backward.  With a position's channels c = 0 .. C-1:
//
//   z = post(y)             post(y)_c = (y_c - mu) rho w_c + b_c,  rho = 1 / sqrt(mean (y - mu)^2 + eps)
//   u = scale * act(gate)   act: identity, sigmoid or silu; gate per sample or per element
//   r = x + u z             the residual stream
//   n = pre(r)              the next block's input
//
// (mu = 0 for the RMS kind, the mean for the layer kind.)  With gradients dr, dn of r and n, and
// h = (y - mu) rho, k = (r - mu') rho':
//
//   t  = dr + rho' (dn w' - mean(dn w') - k mean(dn w' k))        the gradient of r, and of x
//   dz = t u,  dy = rho (dz w - mean(dz w) - h mean(dz w h)),  dgate = t scale z act'(gate)
//   dw' = sum dn k,  db' = sum dn,  dw = sum dz h,  db = sum dz,  dscale = sum t act(gate) z
//
// (the mean(dn w') and mean(dz w) terms only in the layer kind).  Statistics, sums and everything
// between load and store are fp32; r and n are rounded to their type once, n from the unrounded r.
// The backward recomputes r from x and y, so it differentiates what the forward computed.
//
// A forward has to read x, y (and a gate per element) and write r, n; a backward has to read x, y,
// gate, dr, dn and write dx, dy, dgate: about 3 operations per byte, bound by HBM.
#include <algorithm>
#include <cmath>

#include "scx.h"
#include "scx_internal.h"
#include "scx_residual_norm.cuh"

namespace {

using namespace scx_rn;

// ---------------------------------------------------------------------------- any shape
//
// These kernels take any channel count in either layout: TP positions x TC channel threads per
// block, the contiguous axis on neighbouring threads, and a loop over the channels per reduction
// that reads the tensors again (from L1 or L2).

constexpr int kAnyThreads = 256;

struct Split {
    int tp, tc;  // tp * tc = kAnyThreads, powers of two
};

struct Place {
    int p, c;
};

__device__ __forceinline__ Place place_of(const Split& s, bool channels_last) {
    const int t = threadIdx.x;
    return channels_last ? Place{t / s.tc, t % s.tc} : Place{t % s.tp, t / s.tp};
}

// Sums a and b over the channel threads of each position; the same bits in all of them.
__device__ float2 sum_channels(float a, float b, const Split& s, const Place& at) {
    __shared__ float2 red[kAnyThreads];
    float2* row = red + at.p * s.tc;
    __syncthreads();
    row[at.c] = make_float2(a, b);
    for (int o = s.tc / 2; o > 0; o >>= 1) {
        __syncthreads();
        if (at.c < o) {
            row[at.c].x += row[at.c + o].x;
            row[at.c].y += row[at.c + o].y;
        }
    }
    __syncthreads();
    return row[0];
}

__device__ __forceinline__ size_t first_element(const Problem& p, long long q) {
    return p.channels_last ? static_cast<size_t>(q) * p.channels
                           : static_cast<size_t>(q / p.length) * p.channels * p.length + q % p.length;
}

__device__ __forceinline__ size_t channel_stride(const Problem& p) {
    return p.channels_last ? 1 : static_cast<size_t>(p.length);
}

// What the forward computes of one element, given its position's post statistics.
template <typename T>
struct Element {
    float h, z, a, slope, scale, x, r;

    __device__ __forceinline__ Element(const Problem& p, size_t e, long long sample, int c, float mean, float rho) {
        x = to_f32(static_cast<const T*>(p.x)[e]);
        r = x;
        h = z = 0.f;
        a = slope = scale = 1.f;
        if (p.y == nullptr) return;
        const float y = to_f32(static_cast<const T*>(p.y)[e]);
        h = p.post ? (y - mean) * rho : y;
        z = p.post ? fmaf(h, weight<T>(p.post_w, c, p.wide, 1.f), weight<T>(p.post_b, c, p.wide, 0.f)) : y;
        scale = p.scale * weight<T>(p.scale_w, c, p.wide, 1.f);
        if (p.gate_mode != kGateNone) {
            const size_t g = p.gate_mode == kGateFull ? e : static_cast<size_t>(sample) * p.channels + c;
            a = activate(to_f32(static_cast<const T*>(p.gate)[g]), p.act, slope);
        }
        r = fmaf(scale * a, z, x);
    }
};

template <typename T>
__global__ void __launch_bounds__(kAnyThreads) any_forward_kernel(const __grid_constant__ Problem p, Split s) {
    const Place at = place_of(s, p.channels_last);
    const size_t sc = channel_stride(p);
    for (long long q0 = static_cast<long long>(blockIdx.x) * s.tp; q0 < p.positions;
         q0 += static_cast<long long>(gridDim.x) * s.tp) {
        const long long q = q0 + at.p;
        const bool live = q < p.positions;
        const size_t base = live ? first_element(p, q) : 0;
        const long long sample = live ? q / p.length : 0;
        const int end = live ? p.channels : 0;
        float mean = 0.f, rho = 1.f, mean2 = 0.f, rho2 = 1.f;
        if (p.y != nullptr && p.post) {
            const T* y = static_cast<const T*>(p.y);
            float a = 0.f;
            if (p.kind == kLayer) {
                for (int c = at.c; c < end; c += s.tc) a += to_f32(y[base + c * sc]);
                mean = sum_channels(a, 0.f, s, at).x * p.inv_c;
                a = 0.f;
            }
            for (int c = at.c; c < end; c += s.tc) {
                const float d = to_f32(y[base + c * sc]) - mean;
                a = fmaf(d, d, a);
            }
            rho = 1.f / sqrtf(fmaf(sum_channels(a, 0.f, s, at).x, p.inv_c, p.eps));
        }
        if (p.pre) {
            float a = 0.f;
            if (p.kind == kLayer) {
                for (int c = at.c; c < end; c += s.tc) a += Element<T>(p, base + c * sc, sample, c, mean, rho).r;
                mean2 = sum_channels(a, 0.f, s, at).x * p.inv_c;
                a = 0.f;
            }
            for (int c = at.c; c < end; c += s.tc) {
                const float d = Element<T>(p, base + c * sc, sample, c, mean, rho).r - mean2;
                a = fmaf(d, d, a);
            }
            rho2 = 1.f / sqrtf(fmaf(sum_channels(a, 0.f, s, at).x, p.inv_c, p.eps));
        }
        for (int c = at.c; c < end; c += s.tc) {
            const size_t e = base + c * sc;
            const float r = Element<T>(p, e, sample, c, mean, rho).r;
            if (p.r) from_f32(static_cast<T*>(p.r)[e], r);
            if (p.pre)
                from_f32(static_cast<T*>(p.n)[e], fmaf((r - mean2) * rho2, weight<T>(p.pre_w, c, p.wide, 1.f),
                                                       weight<T>(p.pre_b, c, p.wide, 0.f)));
        }
        if (live && at.c == 0 && p.stats) {
            if (p.channels_last) {
                reinterpret_cast<float4*>(p.stats)[q] = make_float4(mean, rho, mean2, rho2);
            } else {
                p.stats[q] = mean;
                p.stats[p.positions + q] = rho;
                p.stats[2 * p.positions + q] = mean2;
                p.stats[3 * p.positions + q] = rho2;
            }
        }
    }
}

struct RowStats {
    float mean, rho, mean2, rho2;
    __device__ __forceinline__ RowStats(const Problem& p, long long q) {
        const float4 s = p.channels_last ? reinterpret_cast<const float4*>(p.stats)[q]
                                         : make_float4(p.stats[q], p.stats[p.positions + q], p.stats[2 * p.positions + q],
                                                       p.stats[3 * p.positions + q]);
        mean = s.x;
        rho = s.y;
        mean2 = s.z;
        rho2 = s.w;
    }
};

template <typename T>
__device__ __forceinline__ float load_or_zero(const void* v, size_t e) {
    return v ? to_f32(static_cast<const T*>(v)[e]) : 0.f;
}

// dx, dy and the gate's gradient per element; leaves the two means of each position for the sums.
template <typename T>
__global__ void __launch_bounds__(kAnyThreads) any_backward_kernel(const __grid_constant__ Problem p, Split s) {
    const Place at = place_of(s, p.channels_last);
    const size_t sc = channel_stride(p);
    for (long long q0 = static_cast<long long>(blockIdx.x) * s.tp; q0 < p.positions;
         q0 += static_cast<long long>(gridDim.x) * s.tp) {
        const long long q = q0 + at.p;
        const bool live = q < p.positions;
        const size_t base = live ? first_element(p, q) : 0;
        const long long sample = live ? q / p.length : 0;
        const int end = live ? p.channels : 0;
        const RowStats st(p, live ? q : 0);
        float m1 = 0.f, m2 = 0.f;
        if (p.dn) {
            float a = 0.f, b = 0.f;
            for (int c = at.c; c < end; c += s.tc) {
                const size_t e = base + c * sc;
                const float r = Element<T>(p, e, sample, c, st.mean, st.rho).r;
                const float d = to_f32(static_cast<const T*>(p.dn)[e]) * weight<T>(p.pre_w, c, p.wide, 1.f);
                a += d;
                b = fmaf(d, (r - st.mean2) * st.rho2, b);
            }
            const float2 m = sum_channels(a, b, s, at);
            m1 = p.kind == kLayer ? m.x * p.inv_c : 0.f;
            m2 = m.y * p.inv_c;
        }
        auto gradient_of_r = [&](const Element<T>& v, size_t e, int c) {
            float t = load_or_zero<T>(p.dr, e);
            if (p.dn) {
                const float d = to_f32(static_cast<const T*>(p.dn)[e]) * weight<T>(p.pre_w, c, p.wide, 1.f);
                t += st.rho2 * (d - m1 - (v.r - st.mean2) * st.rho2 * m2);
            }
            return t;
        };
        float m3 = 0.f, m4 = 0.f;
        if (p.y && p.post && p.dy) {
            float a = 0.f, b = 0.f;
            for (int c = at.c; c < end; c += s.tc) {
                const size_t e = base + c * sc;
                const Element<T> v(p, e, sample, c, st.mean, st.rho);
                const float d = gradient_of_r(v, e, c) * v.scale * v.a * weight<T>(p.post_w, c, p.wide, 1.f);
                a += d;
                b = fmaf(d, v.h, b);
            }
            const float2 m = sum_channels(a, b, s, at);
            m3 = p.kind == kLayer ? m.x * p.inv_c : 0.f;
            m4 = m.y * p.inv_c;
        }
        for (int c = at.c; c < end; c += s.tc) {
            const size_t e = base + c * sc;
            const Element<T> v(p, e, sample, c, st.mean, st.rho);
            const float t = gradient_of_r(v, e, c);
            if (p.dx) from_f32(static_cast<T*>(p.dx)[e], t);
            if (p.dy) {
                const float dz = t * v.scale * v.a;
                from_f32(static_cast<T*>(p.dy)[e],
                         p.post ? st.rho * (dz * weight<T>(p.post_w, c, p.wide, 1.f) - m3 - v.h * m4) : dz);
            }
            if (p.dgate && p.gate_mode == kGateFull)
                from_f32(static_cast<T*>(p.dgate)[e], t * v.scale * v.z * v.slope);
        }
        if (live && at.c == 0 && p.means) {
            p.means[q] = m1;
            p.means[p.positions + q] = m2;
        }
    }
}

// The sums over positions: a block takes one group of tc channels and its share of the tiles (tp
// positions of one sample each).
template <typename T>
__global__ void __launch_bounds__(kAnyThreads) any_sums_kernel(const __grid_constant__ Problem p, Split s) {
    __shared__ float red[kAnyThreads];
    const Place at = place_of(s, p.channels_last);
    const int c = blockIdx.y * s.tc + at.c;
    const bool live = c < p.channels;
    const size_t sc = channel_stride(p);
    auto over_positions = [&](float v) {  // the sum over the positions' threads
        float* column = red + at.c * s.tp;
        __syncthreads();
        column[at.p] = v;
        for (int o = s.tp / 2; o > 0; o >>= 1) {
            __syncthreads();
            if (at.p < o) column[at.p] += column[at.p + o];
        }
        __syncthreads();
        return column[0];
    };
    float sum[kSums] = {};
    long long tile = tile_begin(p, blockIdx.x);
    const long long last = tile_begin(p, blockIdx.x + 1);
    while (tile < last) {
        const long long sample = tile / p.tiles_per_sample;
        const long long stop = min(last, (sample + 1) * p.tiles_per_sample);
        const long long begin = (tile - sample * p.tiles_per_sample) * s.tp;
        const long long end = min(p.length, (stop - sample * p.tiles_per_sample) * s.tp);
        for (long long l = begin + at.p; live && l < end; l += s.tp) {
            const long long q = sample * p.length + l;
            const size_t e = first_element(p, q) + c * sc;
            const RowStats st(p, q);
            const Element<T> v(p, e, sample, c, st.mean, st.rho);
            float t = load_or_zero<T>(p.dr, e);
            if (p.dn) {
                const float dn = to_f32(static_cast<const T*>(p.dn)[e]);
                const float k = (v.r - st.mean2) * st.rho2;
                t += st.rho2 * (dn * weight<T>(p.pre_w, c, p.wide, 1.f) - p.means[q] - k * p.means[p.positions + q]);
                sum[kDPreW] = fmaf(dn, k, sum[kDPreW]);
                sum[kDPreB] += dn;
            }
            const float ta = p.slots ? t : t * v.a;
            sum[kTah] = fmaf(ta, v.h, sum[kTah]);
            sum[kTa] += ta;
        }
        if (p.slots) {
            for (int k = 0; k < 2; ++k) {
                const float total = over_positions(sum[kTah + k]);
                if (live && at.p == 0) slot_of(p, blockIdx.x, sample)[static_cast<size_t>(k) * p.channels + c] = total;
                sum[kTah + k] = 0.f;
            }
        }
        tile = stop;
    }
    for (int k = 0; k < kSums; ++k) {
        const float total = over_positions(sum[k]);
        if (live && at.p == 0)
            p.partial[(static_cast<size_t>(blockIdx.x) * kSums + k) * p.channels + c] = total;
    }
}

// ---------------------------------------------------------------------------- the last sums

constexpr int kFinishThreads = 512;

// Sums over a block's rows, in 64 bits and a fixed order; valid in row 0.
template <int CH>
__device__ double2 sum_rows(double2 v) {
    __shared__ double2 red[kFinishThreads / 32][CH];
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    for (int o = 16; o >= CH; o /= 2) {
        v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
        v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
    }
    __syncthreads();
    if (lane < CH) red[warp][lane] = v;
    __syncthreads();
    if (threadIdx.x < CH) {
        for (int k = 1; k < kFinishThreads / 32; ++k) {
            v.x += red[k][lane].x;
            v.y += red[k][lane].y;
        }
    }
    return v;
}

// Adds the parts' sums per channel, and the slots of each sample into the gradient of its gate.  Grid
// (channels / CH, 2 + samples): y = 0 the norm before the next block, 1 the norm after the block and
// the scale, from 2 on the gates.  Latency is all there is to it, a few hundred rows per channel:
// with few channels, 64 rows of 8 threads keep the chains of loads short (36 channels of 7 samples:
// 7.7 us cold, 12.3 us with 32 rows of 32); with many, whole lines count (2048 channels: 13 us with 8
// threads to a row, 9 us with 32).  The limit of 1024 channels lies between the two that were measured.
template <typename T, int CH>
__global__ void __launch_bounds__(kFinishThreads) finish_kernel(const __grid_constant__ Problem p) {
    constexpr int kFinishRows = kFinishThreads / CH;
    const int row = threadIdx.x / CH;
    const int c = blockIdx.x * CH + threadIdx.x % CH;
    const bool live = c < p.channels;
    const float w = live ? weight<T>(p.post_w, c, p.wide, 1.f) : 0.f, b = live ? weight<T>(p.post_b, c, p.wide, 0.f) : 0.f;
    const float scale = p.scale * (live ? weight<T>(p.scale_w, c, p.wide, 1.f) : 0.f);
    auto add_slot = [&](double2& s, long long part, long long sample, double a) {
        const float* slot = slot_of(p, part, sample) + c;
        s.x += a * slot[0];
        s.y += a * slot[p.channels];
    };
    grid_dep_wait();
    if (blockIdx.y >= 2) {
        for (long long sample = blockIdx.y - 2; sample < p.batch; sample += gridDim.y - 2) {
            double2 s = make_double2(0.0, 0.0);
            const long long last = part_of_tile(p, (sample + 1) * p.tiles_per_sample - 1);
#pragma unroll 4
            for (long long k = part_of_tile(p, sample * p.tiles_per_sample) + row; k <= last; k += kFinishRows)
                if (live) add_slot(s, k, sample, 1.0);
            s = sum_rows<CH>(s);
            if (row != 0 || !live) continue;
            const size_t g = static_cast<size_t>(sample) * p.channels + c;
            float slope;
            activate(to_f32(static_cast<const T*>(p.gate)[g]), p.act, slope);
            from_f32(static_cast<T*>(p.dgate)[g], static_cast<float>(w * s.x + b * s.y) * scale * slope);
        }
        return;
    }
    const bool second = blockIdx.y == 1;
    double2 s = make_double2(0.0, 0.0);
    if (second && p.slots) {
        // the rows share out the samples, as many rows to a sample as there are
        int groups = 1;
        while (groups < kFinishRows && groups < p.batch) groups *= 2;
        const int per_sample = kFinishRows / groups;
        for (long long sample = row / per_sample; live && sample < p.batch; sample += groups) {
            const float a = activate(to_f32(static_cast<const T*>(p.gate)[static_cast<size_t>(sample) * p.channels + c]), p.act);
            const long long last = part_of_tile(p, (sample + 1) * p.tiles_per_sample - 1);
#pragma unroll 4
            for (long long k = part_of_tile(p, sample * p.tiles_per_sample) + row % per_sample; k <= last; k += per_sample)
                add_slot(s, k, sample, a);
        }
    } else if (live) {
        const float* from = p.partial + static_cast<size_t>(second ? kTah : kDPreW) * p.channels + c;
#pragma unroll 8
        for (int k = row; k < p.partials; k += kFinishRows) {
            const float* at = from + static_cast<size_t>(k) * kSums * p.channels;
            s.x += at[0];
            s.y += at[p.channels];
        }
    }
    s = sum_rows<CH>(s);
    if (row != 0 || !live) return;
    if (!second) {
        if (p.d_pre_w) store_weight<T>(p.d_pre_w, c, p.wide, static_cast<float>(s.x));
        if (p.d_pre_b) store_weight<T>(p.d_pre_b, c, p.wide, static_cast<float>(s.y));
    } else {
        if (p.d_post_w) store_weight<T>(p.d_post_w, c, p.wide, static_cast<float>(scale * s.x));
        if (p.d_post_b) store_weight<T>(p.d_post_b, c, p.wide, static_cast<float>(scale * s.y));
        if (p.d_scale) store_weight<T>(p.d_scale, c, p.wide, static_cast<float>(p.scale * (w * s.x + b * s.y)));
    }
}

// ---------------------------------------------------------------------------- host side

constexpr int kMaxChannels = 1 << 18;  // keeps every grid within its limits

Split split_for(const Problem& p) {
    if (!p.channels_last) return {32, kAnyThreads / 32};
    int tc = 1;
    while (tc < p.channels && tc < kAnyThreads) tc *= 2;
    return {kAnyThreads / tc, tc};
}

Split sums_split_for(const Problem& p) {
    return p.channels_last ? Split{kAnyThreads / 32, 32} : Split{32, kAnyThreads / 32};
}

size_t align256(size_t b) { return (b + 255) / 256 * 256; }

struct Layout {
    size_t means, partial, slots, total;
};

Layout layout_of(const scx_residual_norm_config& c) {
    const size_t positions = static_cast<size_t>(c.batch) * static_cast<size_t>(c.length);
    Layout l;
    l.means = 0;
    l.partial = align256(positions * 2 * sizeof(float));
    l.slots = l.partial + align256(static_cast<size_t>(max_parts(c.channels)) * kSums * c.channels * sizeof(float));
    l.total = l.slots;
    if (c.gate_mode == kGateSample)
        l.total += align256((static_cast<size_t>(max_parts(c.channels)) + static_cast<size_t>(c.batch)) * 2 * c.channels * sizeof(float));
    return l;
}

bool valid_config(const scx_residual_norm_config* c) {
    if (!c || c->batch < 0 || c->length < 0 || c->channels <= 0 || c->channels > kMaxChannels) return false;
    if (c->batch > (1LL << 40) || c->length > (1LL << 40)) return false;
    const long long positions = c->batch == 0 ? 0 : (c->length > (1LL << 40) / c->batch ? -1 : c->batch * c->length);
    if (positions < 0 || positions > (1LL << 46) / c->channels) return false;
    return c->channels_last >= 0 && c->channels_last <= 1 && c->dtype >= kF32 && c->dtype <= kF16 &&
           (c->weight_dtype == kF32 || c->weight_dtype == c->dtype) && c->kind >= kRms && c->kind <= kLayer &&
           c->gate_mode >= kGateNone && c->gate_mode <= kGateFull && c->gate_act >= kActNone &&
           c->gate_act <= kActSilu && c->eps >= 0.f && std::isfinite(c->eps) && std::isfinite(c->scale);
}

size_t element_size(int dtype) { return dtype == kF32 ? 4 : 2; }

bool valid_pointer(const void* p, int dtype, bool needed) {
    return p ? reinterpret_cast<uintptr_t>(p) % element_size(dtype) == 0 : !needed;
}

Problem problem_of(const scx_residual_norm_config& c, const scx_residual_norm_tensors& t) {
    Problem p = {};
    p.batch = c.batch;
    p.length = c.length;
    p.positions = c.batch * c.length;
    p.channels = c.channels;
    p.channels_last = c.channels_last;
    p.kind = c.kind;
    p.gate_mode = t.y ? c.gate_mode : kGateNone;
    p.act = c.gate_act;
    p.post = c.post_norm != 0 && t.y != nullptr;
    p.pre = c.pre_norm != 0;
    p.wide = c.weight_dtype == kF32;
    p.eps = c.eps;
    p.inv_c = 1.f / static_cast<float>(c.channels);
    p.scale = c.scale;
    p.x = t.x;
    p.y = t.y;
    p.gate = t.gate;
    // weights of a norm that is not taken are not read by any kernel, nor by the last sums
    p.post_w = p.post ? t.post_weight : nullptr;
    p.post_b = p.post ? t.post_bias : nullptr;
    p.pre_w = p.pre ? t.pre_weight : nullptr;
    p.pre_b = p.pre ? t.pre_bias : nullptr;
    p.scale_w = t.scale;
    p.r = t.r;
    p.n = t.n;
    p.stats = t.stats;
    // the same memory under a simpler description: one position per sample makes the layouts and the
    // gates one; without a gate per sample, tokens do not know of samples
    if (p.length == 1) {
        p.channels_last = 1;
        if (p.gate_mode == kGateSample) p.gate_mode = kGateFull;
    }
    if (p.channels_last && p.gate_mode != kGateSample) {
        p.batch = 1;
        p.length = p.positions;
    }
    return p;
}

bool valid_inputs(const scx_residual_norm_config& c, const scx_residual_norm_tensors& t) {
    return valid_pointer(t.x, c.dtype, true) && valid_pointer(t.y, c.dtype, false) &&
           valid_pointer(t.gate, c.dtype, c.gate_mode != kGateNone && t.y) &&
           valid_pointer(t.post_weight, c.weight_dtype, false) && valid_pointer(t.post_bias, c.weight_dtype, false) &&
           valid_pointer(t.pre_weight, c.weight_dtype, false) && valid_pointer(t.pre_bias, c.weight_dtype, false) &&
           valid_pointer(t.scale, c.weight_dtype, false);
}

int grid_for(long long work) {
    return static_cast<int>(std::max(1LL, std::min(work, static_cast<long long>(scx::num_sms()) * 8)));
}

template <typename T>
cudaError_t forward(const Problem& p, cudaStream_t s) {
    const cudaError_t e = p.channels_last ? token_forward<T>(p, s) : field_forward<T>(p, s);
    if (e != cudaErrorNotSupported) return e;
    const Split split = split_for(p);
    any_forward_kernel<T><<<grid_for((p.positions + split.tp - 1) / split.tp), kAnyThreads, 0, s>>>(p, split);
    return cudaGetLastError();
}

template <typename T>
cudaError_t any_backward(Problem& p, cudaStream_t s) {
    const Split split = split_for(p);
    any_backward_kernel<T><<<grid_for((p.positions + split.tp - 1) / split.tp), kAnyThreads, 0, s>>>(p, split);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess || !p.sums) return e;
    const Split sums = sums_split_for(p);
    p.tiles_per_sample = (p.length + sums.tp - 1) / sums.tp;
    p.tiles = p.batch * p.tiles_per_sample;
    p.parts = static_cast<int>(std::min<long long>(std::min(max_parts(p.channels), 512), p.tiles));
    p.partials = p.parts;
    any_sums_kernel<T><<<dim3(p.parts, (p.channels + sums.tc - 1) / sums.tc), kAnyThreads, 0, s>>>(p, sums);
    return cudaGetLastError();
}

template <typename T>
cudaError_t backward(Problem& p, cudaStream_t s) {
    cudaError_t e = p.channels_last ? token_backward<T>(p, s) : field_backward<T>(p, s);
    if (e == cudaErrorNotSupported) e = any_backward<T>(p, s);
    if (e != cudaSuccess || !p.sums) return e;
    const int gates = p.slots && p.dgate ? static_cast<int>(std::min<long long>(p.batch, 1024)) : 0;
    const bool many = p.channels >= 1024;
    const int ch = many ? 32 : 8;
    return scx::launch_chained(many ? finish_kernel<T, 32> : finish_kernel<T, 8>,
                               dim3((p.channels + ch - 1) / ch, 2 + gates), dim3(kFinishThreads), 0, s, p);
}

}  // namespace

extern "C" int scx_residual_norm_fwd(const scx_residual_norm_config* cfg, const scx_residual_norm_tensors* t,
                                     scx_stream_t stream) {
    if (!valid_config(cfg) || !t) return cudaErrorInvalidValue;
    if (cfg->batch == 0 || cfg->length == 0) return cudaSuccess;
    if (!valid_inputs(*cfg, *t) || !valid_pointer(t->r, cfg->dtype, t->y != nullptr) ||
        !valid_pointer(t->n, cfg->dtype, cfg->pre_norm != 0) || !aligned(t->stats, 16))
        return cudaErrorInvalidValue;
    Problem p = problem_of(*cfg, *t);
    if (!p.y) p.r = nullptr;  // r is x
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    try {
        if (cfg->dtype == kF32) return forward<float>(p, s);
        return cfg->dtype == kBf16 ? forward<__nv_bfloat16>(p, s) : forward<__half>(p, s);
    } catch (...) {
        return cudaErrorMemoryAllocation;
    }
}

extern "C" size_t scx_residual_norm_bwd_workspace_size(const scx_residual_norm_config* cfg) {
    return valid_config(cfg) && cfg->batch > 0 && cfg->length > 0 ? layout_of(*cfg).total : 0;
}

extern "C" int scx_residual_norm_bwd(const scx_residual_norm_config* cfg, const scx_residual_norm_tensors* t,
                                     const scx_residual_norm_grads* g, void* workspace, size_t workspace_bytes,
                                     scx_stream_t stream) {
    if (!valid_config(cfg) || !t || !g || cfg->batch == 0 || cfg->length == 0) return cudaErrorInvalidValue;
    if (!valid_inputs(*cfg, *t) || t->stats == nullptr || !aligned(t->stats, 16) || !valid_pointer(g->dr, cfg->dtype, false) ||
        !valid_pointer(g->dn, cfg->dtype, false) || !valid_pointer(g->dx, cfg->dtype, false) ||
        !valid_pointer(g->dy, cfg->dtype, false) || !valid_pointer(g->dgate, cfg->dtype, false) ||
        !valid_pointer(g->d_post_weight, cfg->weight_dtype, false) ||
        !valid_pointer(g->d_post_bias, cfg->weight_dtype, false) ||
        !valid_pointer(g->d_pre_weight, cfg->weight_dtype, false) ||
        !valid_pointer(g->d_pre_bias, cfg->weight_dtype, false) ||
        !valid_pointer(g->d_scale, cfg->weight_dtype, false) || workspace == nullptr ||
        reinterpret_cast<uintptr_t>(workspace) % 16 != 0 || workspace_bytes < layout_of(*cfg).total)
        return cudaErrorInvalidValue;
    // a gradient of what the forward did not have would be left unwritten
    if ((!t->y && (g->dy || g->dgate || g->d_post_weight || g->d_post_bias || g->d_scale)) ||
        (cfg->gate_mode == kGateNone && g->dgate) || (!cfg->post_norm && (g->d_post_weight || g->d_post_bias)) ||
        (!cfg->pre_norm && (g->dn || g->d_pre_weight || g->d_pre_bias)))
        return cudaErrorInvalidValue;
    Problem p = problem_of(*cfg, *t);
    p.dr = g->dr;
    p.dn = p.pre ? g->dn : nullptr;
    p.dx = g->dx;
    p.dy = p.y ? g->dy : nullptr;
    p.dgate = p.gate_mode != kGateNone ? g->dgate : nullptr;
    p.d_post_w = p.post ? g->d_post_weight : nullptr;
    p.d_post_b = p.post ? g->d_post_bias : nullptr;
    p.d_pre_w = p.pre ? g->d_pre_weight : nullptr;
    p.d_pre_b = p.pre ? g->d_pre_bias : nullptr;
    p.d_scale = p.y ? g->d_scale : nullptr;
    const Layout l = layout_of(*cfg);
    char* ws = static_cast<char*>(workspace);
    p.means = reinterpret_cast<float*>(ws + l.means);
    p.partial = reinterpret_cast<float*>(ws + l.partial);
    const bool of_y = p.d_post_w || p.d_post_b || p.d_scale || (p.gate_mode == kGateSample && p.dgate);
    if (p.gate_mode == kGateSample && of_y) p.slots = reinterpret_cast<float*>(ws + l.slots);
    p.sums = of_y || p.d_pre_w || p.d_pre_b;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    try {
        if (cfg->dtype == kF32) return backward<float>(p, s);
        return cfg->dtype == kBf16 ? backward<__nv_bfloat16>(p, s) : backward<__half>(p, s);
    } catch (...) {
        return cudaErrorMemoryAllocation;
    }
}
