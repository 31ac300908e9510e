// The residual-norm kernels for tokens, [position][channels]: a position's channels are neighbours,
// so 4 to 1024 threads take one position, each NV vectors of VEC channels that stay in registers
// from the first load to the last store; every tensor is read once.  Statistics are sums over a
// position's threads, by shuffles within a warp and through shared memory across warps.
#include <algorithm>

#include "scx_internal.h"
#include "scx_residual_norm.cuh"

namespace scx_rn {
namespace {

constexpr int kMaxThreads = 1024;

// A block of blockDim threads takes blockDim / tpr positions, tpr threads (a power of two) each.
struct Team {
    int tpr, me, row, rows;
    float2* part;  // [2][warps]

    __device__ __forceinline__ Team(int threads, float2* shared)
        : tpr(threads), me(threadIdx.x % threads), row(threadIdx.x / threads), rows(blockDim.x / threads), part(shared) {}

    // Sums over the position's threads, the same bits in all of them.  `turn` alternates between
    // calls, so that one barrier per call is enough.
    __device__ __forceinline__ float2 sum(float a, float b, int& turn) {
        for (int o = min(tpr, 32) / 2; o > 0; o >>= 1) {
            a += __shfl_xor_sync(0xffffffffu, a, o);
            b += __shfl_xor_sync(0xffffffffu, b, o);
        }
        if (tpr <= 32) return make_float2(a, b);
        float2* now = part + turn * (kMaxThreads / 32);
        turn ^= 1;
        if (threadIdx.x % 32 == 0) now[threadIdx.x / 32] = make_float2(a, b);
        __syncthreads();
        const int warps = tpr / 32;
        const float2* mine = now + row * warps;
        float2 s = mine[0];
        for (int w = 1; w < warps; ++w) {
            s.x += mine[w].x;
            s.y += mine[w].y;
        }
        return s;
    }
};

template <typename T, int VEC>
__device__ __forceinline__ void weights(const void* w, int c, bool live, bool wide, float other, float (&out)[VEC]) {
    if (w == nullptr || !live) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) out[i] = other;
    } else if (wide) {
        constexpr int kPer = VEC < 4 ? VEC : 4;
#pragma unroll
        for (int i = 0; i < VEC; i += kPer) {
            const Vec<float, kPer> v = load_vec<float, kPer>(w, c + i);
#pragma unroll
            for (int k = 0; k < kPer; ++k) out[i + k] = v.v[k];
        }
    } else {
        const Vec<T, VEC> v = load_vec<T, VEC>(w, c);
#pragma unroll
        for (int i = 0; i < VEC; ++i) out[i] = to_f32(v.v[i]);
    }
}

// Mean and 1 / sqrt(variance + eps) of a position's values.
template <int VEC, int NV>
__device__ __forceinline__ float2 statistics(const Problem& p, Team& team, const float (&v)[NV][VEC],
                                             const bool (&live)[NV], int& turn) {
    float mean = 0.f, s = 0.f;
    if (p.kind == kLayer) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < VEC; ++i) s += live[j] ? v[j][i] : 0.f;
        mean = team.sum(s, 0.f, turn).x * p.inv_c;
        s = 0.f;
    }
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const float d = live[j] ? v[j][i] - mean : 0.f;
            s = fmaf(d, d, s);
        }
    return make_float2(mean, 1.f / sqrtf(fmaf(team.sum(s, 0.f, turn).x, p.inv_c, p.eps)));
}

template <typename T, int VEC, int NV>
__global__ void __launch_bounds__(kMaxThreads) token_forward_kernel(const __grid_constant__ Problem p, int tpr) {
    __shared__ float2 part[2 * kMaxThreads / 32];
    Team team(tpr, part);
    int turn = 0;
    for (long long q0 = static_cast<long long>(blockIdx.x) * team.rows; q0 < p.positions;
         q0 += static_cast<long long>(gridDim.x) * team.rows) {
        const long long q = q0 + team.row;
        const size_t base = static_cast<size_t>(q) * p.channels;
        const size_t gate = p.gate_mode == kGateSample ? static_cast<size_t>(q / p.length) * p.channels : base;
        Vec<T, VEC> x[NV], y[NV], g[NV];
        bool live[NV];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * tpr + team.me) * VEC;
            live[j] = q < p.positions && c < p.channels;
            x[j] = y[j] = g[j] = Vec<T, VEC>{};
            if (live[j]) {
                x[j] = load_vec<T, VEC>(p.x, base + c);
                if (p.y) y[j] = load_vec<T, VEC>(p.y, base + c);
                if (p.gate_mode != kGateNone) g[j] = load_vec<T, VEC>(p.gate, gate + c);
            }
        }
        float r[NV][VEC];
        float2 st = make_float2(0.f, 1.f), st2 = st;
        if (p.y) {
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int i = 0; i < VEC; ++i) r[j][i] = to_f32(y[j].v[i]);
            if (p.post) st = statistics<VEC, NV>(p, team, r, live, turn);
        }
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * tpr + team.me) * VEC;
            if (p.y) {
                float w[VEC], b[VEC], scale[VEC];
                weights<T, VEC>(p.post_w, c, live[j], p.wide, 1.f, w);
                weights<T, VEC>(p.post_b, c, live[j], p.wide, 0.f, b);
                weights<T, VEC>(p.scale_w, c, live[j], p.wide, 1.f, scale);
                Vec<T, VEC> o;
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const float a = p.gate_mode == kGateNone ? 1.f : activate(to_f32(g[j].v[i]), p.act);
                    const float z = fmaf((r[j][i] - st.x) * st.y, w[i], b[i]);
                    r[j][i] = fmaf(p.scale * scale[i] * a, z, to_f32(x[j].v[i]));
                    from_f32(o.v[i], r[j][i]);
                }
                if (live[j]) store_vec<T, VEC>(p.r, base + c, o);
            } else {
#pragma unroll
                for (int i = 0; i < VEC; ++i) r[j][i] = to_f32(x[j].v[i]);
            }
        }
        if (p.pre) {
            st2 = statistics<VEC, NV>(p, team, r, live, turn);
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int c = (j * tpr + team.me) * VEC;
                float w[VEC], b[VEC];
                weights<T, VEC>(p.pre_w, c, live[j], p.wide, 1.f, w);
                weights<T, VEC>(p.pre_b, c, live[j], p.wide, 0.f, b);
                Vec<T, VEC> o;
#pragma unroll
                for (int i = 0; i < VEC; ++i) from_f32(o.v[i], fmaf((r[j][i] - st2.x) * st2.y, w[i], b[i]));
                if (live[j]) store_vec<T, VEC>(p.n, base + c, o);
            }
        }
        if (p.stats && team.me == 0 && q < p.positions) {
            p.stats[q] = st.x;
            p.stats[p.positions + q] = st.y;
            p.stats[2 * p.positions + q] = st2.x;
            p.stats[3 * p.positions + q] = st2.y;
        }
    }
}

// Sums over a block's positions: the rows' threads of one channel are added through shared memory in
// row order, and row 0 stores the result.
template <int VEC, int NV>
__device__ void store_sums(const Problem& p, const Team& team, float* shared, const float (&sum)[NV][VEC], float* out) {
    __syncthreads();
    if (team.rows > 1) {
        const int width = team.tpr * VEC * NV;
        for (int j = 0; j < NV; ++j)
            for (int i = 0; i < VEC; ++i) shared[team.row * width + (j * team.tpr + team.me) * VEC + i] = sum[j][i];
        __syncthreads();
        for (int c = threadIdx.x; c < p.channels; c += blockDim.x) {
            float s = 0.f;
            for (int r = 0; r < team.rows; ++r) s += shared[r * width + c];
            out[c] = s;
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = (j * team.tpr + team.me) * VEC;
#pragma unroll
        for (int i = 0; i < VEC; ++i)
            if (c + i < p.channels) out[c + i] = sum[j][i];
    }
}

template <typename T, int VEC, int NV>
__global__ void __launch_bounds__(512) token_backward_kernel(const __grid_constant__ Problem p, int tpr) {
    extern __shared__ float shared[];  // the rows' sums; unused where a block has one row
    __shared__ float2 part[2 * kMaxThreads / 32];
    grid_dep_launch();
    Team team(tpr, part);
    int turn = 0;
    float dw2[NV][VEC] = {}, db2[NV][VEC] = {}, tah[NV][VEC] = {}, ta[NV][VEC] = {};
    const long long last = tile_begin(p, blockIdx.x + 1);
    for (long long tile = tile_begin(p, blockIdx.x); tile < last; ++tile) {
        const long long sample = p.tiles_per_sample == p.tiles ? 0 : tile / p.tiles_per_sample;
        const long long l = (tile - sample * p.tiles_per_sample) * team.rows + team.row;
        const bool here = l < p.length;
        const long long q = sample * p.length + (here ? l : 0);
        const size_t base = static_cast<size_t>(q) * p.channels;
        const size_t gate = p.gate_mode == kGateSample ? static_cast<size_t>(sample) * p.channels : base;
        Vec<T, VEC> x[NV], y[NV], g[NV], dr[NV], dn[NV];
        bool live[NV];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * tpr + team.me) * VEC;
            live[j] = here && c < p.channels;
            x[j] = y[j] = g[j] = dr[j] = dn[j] = Vec<T, VEC>{};
            if (live[j]) {
                if (p.dn) x[j] = load_vec<T, VEC>(p.x, base + c);
                if (p.y) y[j] = load_vec<T, VEC>(p.y, base + c);
                if (p.gate_mode != kGateNone) g[j] = load_vec<T, VEC>(p.gate, gate + c);
                if (p.dr) dr[j] = load_vec<T, VEC>(p.dr, base + c);
                if (p.dn) dn[j] = load_vec<T, VEC>(p.dn, base + c);
            }
        }
        const float mean = p.post ? p.stats[q] : 0.f, rho = p.post ? p.stats[p.positions + q] : 1.f;
        const float mean2 = p.pre ? p.stats[2 * p.positions + q] : 0.f, rho2 = p.pre ? p.stats[3 * p.positions + q] : 0.f;
        float h[NV][VEC], k[NV][VEC], t[NV][VEC], a[NV][VEC];
        float s0 = 0.f, s1 = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * tpr + team.me) * VEC;
            float w[VEC], b[VEC], scale[VEC], w2[VEC];
            weights<T, VEC>(p.post_w, c, live[j], p.wide, 1.f, w);
            weights<T, VEC>(p.post_b, c, live[j], p.wide, 0.f, b);
            weights<T, VEC>(p.scale_w, c, live[j], p.wide, 1.f, scale);
            weights<T, VEC>(p.pre_w, c, live[j], p.wide, 1.f, w2);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const bool on = live[j];
                a[j][i] = p.gate_mode == kGateNone ? 1.f : activate(to_f32(g[j].v[i]), p.act);
                h[j][i] = p.y && on ? (to_f32(y[j].v[i]) - mean) * rho : 0.f;
                const float r = fmaf(p.scale * scale[i] * a[j][i], p.y ? fmaf(h[j][i], w[i], b[i]) : 0.f, to_f32(x[j].v[i]));
                k[j][i] = (r - mean2) * rho2;
                const float n = to_f32(dn[j].v[i]);  // zero where not live
                t[j][i] = n * w2[i];
                s0 += t[j][i];
                s1 = fmaf(t[j][i], k[j][i], s1);
                dw2[j][i] = fmaf(n, k[j][i], dw2[j][i]);
                db2[j][i] += n;
            }
        }
        float2 m = make_float2(0.f, 0.f);
        if (p.dn) {
            m = team.sum(s0, s1, turn);
            m.x = p.kind == kLayer ? m.x * p.inv_c : 0.f;
            m.y *= p.inv_c;
        }
        s0 = s1 = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * tpr + team.me) * VEC;
            float w[VEC], scale[VEC];
            weights<T, VEC>(p.post_w, c, live[j], p.wide, 1.f, w);
            weights<T, VEC>(p.scale_w, c, live[j], p.wide, 1.f, scale);
            Vec<T, VEC> o;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                t[j][i] = live[j] ? to_f32(dr[j].v[i]) + rho2 * (t[j][i] - m.x - k[j][i] * m.y) : 0.f;
                from_f32(o.v[i], t[j][i]);
                const float d = t[j][i] * a[j][i] * (p.scale * scale[i] * w[i]);
                s0 += d;
                s1 = fmaf(d, h[j][i], s1);
                const float v = p.slots ? t[j][i] : t[j][i] * a[j][i];
                tah[j][i] = fmaf(v, h[j][i], tah[j][i]);
                ta[j][i] += v;
            }
            if (p.dx && live[j]) store_vec<T, VEC>(p.dx, base + c, o);
        }
        float2 m2 = make_float2(0.f, 0.f);
        if (p.post && p.dy) {
            m2 = team.sum(s0, s1, turn);
            m2.x = p.kind == kLayer ? m2.x * p.inv_c : 0.f;
            m2.y *= p.inv_c;
        }
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * tpr + team.me) * VEC;
            float w[VEC], b[VEC], scale[VEC];
            weights<T, VEC>(p.post_w, c, live[j], p.wide, 1.f, w);
            weights<T, VEC>(p.post_b, c, live[j], p.wide, 0.f, b);
            weights<T, VEC>(p.scale_w, c, live[j], p.wide, 1.f, scale);
            Vec<T, VEC> o;
            if (p.dy) {
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const float d = t[j][i] * a[j][i] * (p.scale * scale[i] * w[i]);
                    from_f32(o.v[i], p.post ? rho * (d - m2.x - h[j][i] * m2.y) : d);
                }
                if (live[j]) store_vec<T, VEC>(p.dy, base + c, o);
            }
            if (p.dgate && p.gate_mode == kGateFull) {
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    float slope;
                    activate(to_f32(g[j].v[i]), p.act, slope);
                    from_f32(o.v[i], t[j][i] * (p.scale * scale[i]) * fmaf(h[j][i], w[i], b[i]) * slope);
                }
                if (live[j]) store_vec<T, VEC>(p.dgate, base + c, o);
            }
        }
        if (p.slots && (tile + 1 == last || (tile + 1) % p.tiles_per_sample == 0)) {
            float* slot = slot_of(p, blockIdx.x, sample);
            store_sums<VEC, NV>(p, team, shared, tah, slot);
            store_sums<VEC, NV>(p, team, shared, ta, slot + p.channels);
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int i = 0; i < VEC; ++i) tah[j][i] = ta[j][i] = 0.f;
        }
    }
    if (!p.sums) return;
    float* out = p.partial + static_cast<size_t>(blockIdx.x) * kSums * p.channels;
    store_sums<VEC, NV>(p, team, shared, dw2, out + static_cast<size_t>(kDPreW) * p.channels);
    store_sums<VEC, NV>(p, team, shared, db2, out + static_cast<size_t>(kDPreB) * p.channels);
    store_sums<VEC, NV>(p, team, shared, tah, out + static_cast<size_t>(kTah) * p.channels);
    store_sums<VEC, NV>(p, team, shared, ta, out + static_cast<size_t>(kTa) * p.channels);
}

// Threads per position: a power of two that covers the channels.
int team_for(int channels, int per_thread) {
    int tpr = 4;
    while (tpr * per_thread < channels) tpr *= 2;
    return tpr;
}

template <typename T, int VEC, int NV>
cudaError_t forward_as(const Problem& p, cudaStream_t s) {
    const int tpr = team_for(p.channels, VEC * NV);
    const int threads = std::max(128, tpr), rows = threads / tpr;
    const long long blocks = (p.positions + rows - 1) / rows;
    const int grid = static_cast<int>(std::min<long long>(blocks, 64LL * scx::num_sms()));
    token_forward_kernel<T, VEC, NV><<<grid, threads, 0, s>>>(p, tpr);
    return cudaGetLastError();
}

template <typename T, int VEC, int NV>
cudaError_t backward_as(Problem& p, cudaStream_t s) {
    const int tpr = team_for(p.channels, VEC * NV);
    const int threads = std::max(128, tpr), rows = threads / tpr;
    const size_t smem = rows > 1 ? sizeof(float) * threads * VEC * NV : 0;
    int per_sm = 0;
    const cudaError_t e =
        scx::prepare_kernel(reinterpret_cast<const void*>(token_backward_kernel<T, VEC, NV>), smem, threads, &per_sm);
    if (e != cudaSuccess) return e;
    p.tiles_per_sample = (p.length + rows - 1) / rows;
    p.tiles = p.batch * p.tiles_per_sample;
    p.parts = static_cast<int>(std::min<long long>(std::min(max_parts(p.channels), per_sm * scx::num_sms()), p.tiles));
    token_backward_kernel<T, VEC, NV><<<p.parts, threads, smem, s>>>(p, tpr);
    return cudaGetLastError();
}

// Whether rows can be moved by 16-byte accesses: whole vectors per row, every base aligned.
template <typename T>
bool vectors_fit(const Problem& p) {
    const void* all[] = {p.x, p.y, p.gate_mode != kGateNone ? p.gate : nullptr, p.r, p.n, p.dr, p.dn, p.dx, p.dy,
                         p.gate_mode == kGateFull ? p.dgate : nullptr, p.post_w, p.post_b, p.pre_w, p.pre_b, p.scale_w};
    for (const void* a : all)
        if (!aligned(a, 16)) return false;
    return p.channels % (16 / static_cast<int>(sizeof(T))) == 0;
}

}  // namespace

template <typename T>
cudaError_t token_forward(const Problem& p, cudaStream_t s) {
    constexpr int VEC = 16 / static_cast<int>(sizeof(T));
    if (vectors_fit<T>(p)) {
        if (p.channels <= VEC * 1024) return forward_as<T, VEC, 1>(p, s);
        if (p.channels <= 2 * VEC * 1024) return forward_as<T, VEC, 2>(p, s);
        return cudaErrorNotSupported;
    }
    if (p.channels <= 2048) return forward_as<T, 1, 4>(p, s);
    if (p.channels <= 8192) return forward_as<T, 1, 8>(p, s);
    return cudaErrorNotSupported;
}

template <typename T>
cudaError_t token_backward(Problem& p, cudaStream_t s) {
    constexpr int VEC = 16 / static_cast<int>(sizeof(T));
    if (vectors_fit<T>(p)) {
        if (p.channels <= VEC * 512) return backward_as<T, VEC, 1>(p, s);
        if (sizeof(T) == 4 && p.channels <= 2 * VEC * 512) return backward_as<T, VEC, sizeof(T) == 4 ? 2 : 1>(p, s);
        return cudaErrorNotSupported;
    }
    if (p.channels <= 2048) return backward_as<T, 1, 4>(p, s);
    return cudaErrorNotSupported;
}

template cudaError_t token_forward<float>(const Problem&, cudaStream_t);
template cudaError_t token_forward<__nv_bfloat16>(const Problem&, cudaStream_t);
template cudaError_t token_forward<__half>(const Problem&, cudaStream_t);
template cudaError_t token_backward<float>(Problem&, cudaStream_t);
template cudaError_t token_backward<__nv_bfloat16>(Problem&, cudaStream_t);
template cudaError_t token_backward<__half>(Problem&, cudaStream_t);

}  // namespace scx_rn
