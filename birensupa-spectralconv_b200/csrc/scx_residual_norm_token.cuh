// The residual-norm kernels for tokens, [position][channels]: a position's channels are neighbours,
// so 4 to 512 threads take one position, each NV vectors of VEC channels, and every tensor is read
// once: the values of the next positions are copied into the thread's own slots in shared memory
// while this one's are in registers.  A thread keeps its channels from position to position, with
// their weights, and in the backward their sums, in registers.  Statistics are sums over a
// position's threads, by shuffles within a warp and through shared memory across warps.
//
// What a thread keeps bounds a block to 512 threads and 8 or 16 channels per thread.  Longer
// positions are cut over a cluster of CL = 2 or 4 blocks, which exchange their parts of each sum through
// distributed shared memory.
#pragma once

#include <algorithm>

#include "scx_internal.h"
#include "scx_residual_norm.cuh"

namespace scx_rn {
namespace {

constexpr int kMaxThreads = 512;
constexpr int kAhead = 2;  // positions whose copies are under way while one is computed
constexpr int kParts = kMaxThreads / 32 * 4 * 2;  // two numbers per warp of a cluster
constexpr int kPartBytes = 2 * kParts * sizeof(float);

__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Writes v to the same place of block `rank`'s shared memory as `at` has in this one's.
__device__ __forceinline__ void store_in_block(float* at, int rank, float v) {
    unsigned to;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
                 : "=r"(to)
                 : "r"(static_cast<unsigned>(__cvta_generic_to_shared(at))), "r"(rank));
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to), "f"(v) : "memory");
}

// A cluster of CL blocks takes blockDim / tpr positions (one, where CL > 1), tpr threads (a power of
// two) of each block to a position.
template <int VEC, int CL>
struct Team {
    int tpr, me, row, rows, rank;
    int first, end;  // this thread's first channel, and where the block's channels end
    float* part;     // [2][kParts]

    __device__ __forceinline__ Team(int threads, int columns, int channels, float* shared)
        : tpr(threads), me(threadIdx.x % threads), row(threadIdx.x / threads), rows(blockDim.x / threads),
          rank(blockIdx.x % CL), first(rank * columns + me * VEC), end(min(channels, (rank + 1) * columns)), part(shared) {
        if (CL > 1) cluster_barrier();  // the others' shared memory is there
    }

    // The first channel of the thread's vector j, and whether it exists.
    __device__ __forceinline__ int channel(int j) const { return first + j * tpr * VEC; }
    __device__ __forceinline__ bool has(int j) const { return channel(j) < end; }

    // Sums K (one or two) numbers over the position's threads, the same bits in all of them.  Two share
    // the steps: after the first, one half of the warp adds the first number and the other the second.
    // Across warps every warp adds the warps' parts itself; `turn` alternates between calls, so that
    // one barrier per call is enough.
    template <int K>
    __device__ __forceinline__ void sum(float (&v)[K], int& turn) {
        const int lane = threadIdx.x % 32;
        if (CL == 1 && tpr < 32) {
            for (int o = tpr / 2; o > 0; o >>= 1) {
#pragma unroll
                for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
            }
            return;
        }
        float s = v[0];
        if (K == 2) {
            const float give = lane < 16 ? v[K - 1] : v[0];
            s = (lane < 16 ? v[0] : v[K - 1]) + __shfl_xor_sync(0xffffffffu, give, 16);
        } else {
            s += __shfl_xor_sync(0xffffffffu, s, 16);
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (CL == 1 && tpr == 32) {
            const float other = K == 2 ? __shfl_xor_sync(0xffffffffu, s, 16) : s;
            v[0] = lane < 16 ? s : other;
            v[K - 1] = lane < 16 ? other : s;
            return;
        }
        // the warps' numbers, K to a warp, in a row; a lane takes every 32nd, so always number lane % K
        constexpr int kMost = kMaxThreads / 32;  // warps of a block
        float* now = part + turn * kParts;
        turn ^= 1;
        const int warp = threadIdx.x / 32;
        if (CL > 1) {
            // to every block of the cluster: one lane per block and number
            const float mine = __shfl_sync(0xffffffffu, s, lane < CL ? 0 : 16);
            if (lane < CL * K) store_in_block(now + (rank * kMost + warp) * K + lane / CL, lane % CL, mine);
            __syncwarp();
            cluster_barrier();
            s = 0.f;
#pragma unroll
            for (int e = 0; e < CL * kMost * K; e += 32) s += now[e + lane];
        } else {
            if (lane % 16 == 0 && lane < 16 * K) now[warp * K + lane / 16] = s;
            __syncthreads();
            const int warps = tpr / 32;  // 2, 4, 8 or 16
            s = lane < warps * K ? now[row * warps * K + lane] : 0.f;
        }
#pragma unroll
        for (int o = 16; o >= K; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (K == 2) {
            const float other = __shfl_xor_sync(0xffffffffu, s, 1);
            v[0] = lane % 2 ? other : s;
            v[K - 1] = lane % 2 ? s : other;
        } else {
            v[0] = s;
        }
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
            for (int k = 0; k < kPer; ++k) out[i + k] = v.w[k];
        }
    } else {
        const Vec<T, VEC> v = load_vec<T, VEC>(w, c);
        if constexpr (VEC == 1) {
            out[0] = v.one();
        } else {
#pragma unroll
            for (int i = 0; i < VEC / 2; ++i) {
                const float2 two = v.pair(i);
                out[2 * i] = two.x;
                out[2 * i + 1] = two.y;
            }
        }
    }
}

// A thread's values lie in pairs of neighbours of its NV * VEC channels.
template <int P>
__device__ __forceinline__ float sum_of(const float2 (&v)[P]) {
    float2 s = v[0];
#pragma unroll
    for (int i = 1; i < P; ++i) s = add2(s, v[i]);
    return s.x + s.y;
}

// Mean and 1 / sqrt(variance + eps) of a position's values; vectors that do not exist hold zeros.
template <int VEC, int NV, typename TEAM>
__device__ __forceinline__ float2 statistics(const Problem& p, TEAM& team, const float2 (&v)[NV * VEC / 2],
                                             const bool (&on)[NV], int& turn) {
    constexpr int P = NV * VEC / 2;
    float mean = 0.f, s[1];
    float2 d[P];
    if (p.kind == kLayer) {
        s[0] = sum_of(v);
        team.sum(s, turn);
        mean = s[0] * p.inv_c;
#pragma unroll
        for (int i = 0; i < P; ++i) {
            d[i] = add2(v[i], both(-mean));
            if (!on[2 * i / VEC]) d[i].x = 0.f;
            if (!on[(2 * i + 1) / VEC]) d[i].y = 0.f;
            d[i] = mul2(d[i], d[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < P; ++i) d[i] = mul2(v[i], v[i]);
    }
    s[0] = sum_of(d);
    team.sum(s, turn);
    return make_float2(mean, rsqrtf(fmaf(s[0], p.inv_c, p.eps)));
}

template <typename T, int VEC, int NV, typename TEAM>
__device__ __forceinline__ void weight_pairs(const void* w, const Problem& p, const TEAM& team, float other,
                                             float2 (&out)[NV * VEC / 2]) {
    float v[NV][VEC];
#pragma unroll
    for (int j = 0; j < NV; ++j) weights<T, VEC>(w, team.channel(j), team.has(j), p.wide, other, v[j]);
#pragma unroll
    for (int i = 0; i < NV * VEC / 2; ++i) out[i] = make_float2(v[2 * i / VEC][2 * i % VEC], v[(2 * i + 1) / VEC][(2 * i + 1) % VEC]);
}

// The weights of a thread's channels, the scale taken into those of the norm after the block.
template <typename T, int VEC, int NV>
struct Weights {
    float2 w[NV * VEC / 2], b[NV * VEC / 2], w2[NV * VEC / 2];

    template <typename TEAM>
    __device__ __forceinline__ Weights(const Problem& p, const TEAM& team, bool block) {
        if (block) {
            float2 scale[NV * VEC / 2];
            weight_pairs<T, VEC, NV>(p.scale_w, p, team, 1.f, scale);
            weight_pairs<T, VEC, NV>(p.post ? p.post_w : nullptr, p, team, 1.f, w);
            weight_pairs<T, VEC, NV>(p.post ? p.post_b : nullptr, p, team, 0.f, b);
#pragma unroll
            for (int i = 0; i < NV * VEC / 2; ++i) {
                scale[i] = mul2(scale[i], both(p.scale));
                w[i] = mul2(w[i], scale[i]);
                b[i] = mul2(b[i], scale[i]);
            }
        }
        weight_pairs<T, VEC, NV>(p.pre_w, p, team, 1.f, w2);
    }
};

// Where a thread's vectors of one position lie in a tensor, in bytes; zero where there is none.
template <int NV>
struct Row {
    size_t at[NV];
    bool live[NV];
};

// A thread's slots in shared memory, and how it fills and reads them: slot k is a tensor of a position
// under way, NV vectors, `pitch` bytes apart.
template <typename T, int VEC, int NV>
struct Slots {
    using E = Vec<T, VEC>;
    unsigned char* base;
    unsigned address, pitch;
    int channel[NV];  // in bytes
    bool on[NV];

    template <typename TEAM>
    __device__ __forceinline__ Slots(unsigned char* shared, const TEAM& team)
        : base(shared + threadIdx.x * sizeof(E)), address(shared_address(base)), pitch(blockDim.x * sizeof(E)) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            on[j] = team.has(j);
            channel[j] = on[j] ? team.channel(j) * static_cast<int>(sizeof(T)) : 0;
        }
    }

    // `first`: the position's first element
    __device__ __forceinline__ Row<NV> row(size_t first, bool here) const {
        Row<NV> r;
        const size_t bytes = here ? first * sizeof(T) : 0;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            r.at[j] = bytes + channel[j];
            r.live[j] = here && on[j];
        }
        return r;
    }

    __device__ __forceinline__ void fetch(unsigned k, const void* from, const Row<NV>& r) const {
        if constexpr (kCopied<E>) {
#pragma unroll
            for (int j = 0; j < NV; ++j)
                copy_async<E>(address + (k * NV + j) * pitch, static_cast<const char*>(from) + r.at[j], r.live[j]);
        }
    }

    __device__ __forceinline__ void read(unsigned k, const void* from, const Row<NV>& r,
                                         float2 (&out)[NV * VEC / 2]) const {
        E v[NV];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            v[j] = E{};
            if constexpr (kCopied<E>) v[j] = *reinterpret_cast<const E*>(base + (k * NV + j) * pitch);
            else if (r.live[j]) v[j] = *reinterpret_cast<const E*>(static_cast<const char*>(from) + r.at[j]);
        }
#pragma unroll
        for (int i = 0; i < NV * VEC / 2; ++i) {
            if constexpr (VEC == 1) out[i] = make_float2(v[2 * i].one(), v[2 * i + 1].one());
            else out[i] = v[2 * i / VEC].pair(i % (VEC / 2));
        }
    }

    __device__ __forceinline__ void store(void* to, const Row<NV>& r, const float2 (&v)[NV * VEC / 2]) const {
        E o[NV];
#pragma unroll
        for (int i = 0; i < NV * VEC / 2; ++i) {
            if constexpr (VEC == 1) {
                o[2 * i].set_one(v[i].x);
                o[2 * i + 1].set_one(v[i].y);
            } else {
                o[2 * i / VEC].set_pair(i % (VEC / 2), v[i]);
            }
        }
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (r.live[j]) *reinterpret_cast<E*>(static_cast<char*>(to) + r.at[j]) = o[j];
    }
};

// Zeros where there is no channel.
template <int VEC, int NV>
__device__ __forceinline__ void clear_dead(float2 (&v)[NV * VEC / 2], const bool (&on)[NV]) {
#pragma unroll
    for (int i = 0; i < NV * VEC / 2; ++i) {
        if (!on[2 * i / VEC]) v[i].x = 0.f;
        if (!on[(2 * i + 1) / VEC]) v[i].y = 0.f;
    }
}

__host__ __device__ constexpr int forward_tensors(int mode) { return mode == kNoBlock ? 1 : mode == kPlain ? 2 : 3; }
__host__ __device__ constexpr int backward_tensors(int mode) { return mode == kNoBlock ? 3 : mode == kPlain ? 4 : 5; }

// A gate per sample is read like one per element, from the sample's row: kSample and kFull are one
// mode here.
template <typename T, int VEC, int NV, int CL, int MODE>
__global__ void __launch_bounds__(kMaxThreads) token_forward_kernel(const __grid_constant__ Problem p, int tpr,
                                                                    int columns) {
    using F = Slots<T, VEC, NV>;
    constexpr int N = NV * VEC / 2, kTensors = forward_tensors(MODE);
    extern __shared__ __align__(16) unsigned char dynamic[];
    auto* part = reinterpret_cast<float*>(dynamic);
    Team<VEC, CL> team(tpr, columns, p.channels, part);
    const int channels = p.channels;
    const long long block = blockIdx.x / CL, blocks = gridDim.x / CL;  // clusters
    const long long groups = (p.positions + team.rows - 1) / team.rows;
    const F slots(dynamic + kPartBytes, team);
    const auto& on = slots.on;
    auto gate_row = [&](long long q, bool here) {
        return slots.row(static_cast<size_t>(p.gate_mode == kGateSample ? q / p.length : q) * channels, here);
    };
    auto fetch = [&](long long group, int ring) {
        if (group < groups) {
            const long long q = group * team.rows + team.row;
            const bool here = q < p.positions;
            const Row<NV> row = slots.row(static_cast<size_t>(q) * channels, here);
            const unsigned k = ring * kTensors;
            slots.fetch(k, p.x, row);
            if constexpr (MODE != kNoBlock) slots.fetch(k + 1, p.y, row);
            if constexpr (MODE == kFull) slots.fetch(k + 2, p.gate, p.gate_mode == kGateSample ? gate_row(q, here) : row);
        }
        copy_commit();
    };
#pragma unroll
    for (int k = 0; k < kAhead; ++k) fetch(block + k * blocks, k);
    const Weights<T, VEC, NV> weight_of(p, team, MODE != kNoBlock);
    int turn = 0, ring = 0;
    for (long long group = block; group < groups; group += blocks) {
        const long long q = group * team.rows + team.row;
        const bool here = q < p.positions;
        const Row<NV> row = slots.row(static_cast<size_t>(q) * channels, here);
        const unsigned slot = ring * kTensors;
        fetch(group + kAhead * blocks, ring == 0 ? kAhead : ring - 1);
        copy_wait<kAhead>();
        float2 r[N], st = make_float2(0.f, 1.f), st2 = st;
        slots.read(slot, p.x, row, r);
        if constexpr (MODE != kNoBlock) {
            float2 h[N], a[N];
            slots.read(slot + 1, p.y, row, h);
            if constexpr (MODE == kFull) {
                slots.read(slot + 2, p.gate, kCopied<typename F::E> ? row : gate_row(q, here), a);
                activate_all<T>(a, p.act);
            }
            if (p.post) st = statistics<VEC, NV>(p, team, h, on, turn);
            const float2 rho = both(st.y), shift = both(-st.x * st.y);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float2 z = fma2(fma2(h[i], rho, shift), weight_of.w[i], weight_of.b[i]);
                r[i] = MODE == kPlain ? add2(r[i], z) : fma2(a[i], z, r[i]);
            }
            slots.store(p.r, row, r);
            clear_dead<VEC, NV>(r, on);
        }
        if (p.pre) {
            st2 = statistics<VEC, NV>(p, team, r, on, turn);
            const float2 rho = both(st2.y), shift = both(-st2.x * st2.y);
            float2 b[N];
            weight_pairs<T, VEC, NV>(p.pre_b, p, team, 0.f, b);
#pragma unroll
            for (int i = 0; i < N; ++i) r[i] = fma2(fma2(r[i], rho, shift), weight_of.w2[i], b[i]);
            slots.store(p.n, row, r);
        }
        if (p.stats && team.rank == 0 && team.me == 0 && here)
            reinterpret_cast<float4*>(p.stats)[q] = make_float4(st.x, st.y, st2.x, st2.y);
        ring = ring == kAhead ? 0 : ring + 1;
    }
    copy_wait<0>();
}

// Sums over a block's positions: the rows' threads of one channel are added through shared memory in
// row order.  Every thread of the block calls it.
template <int VEC, int NV, typename TEAM>
__device__ void store_sums(const Problem& p, const TEAM& team, float* shared, const float2 (&sum)[NV * VEC / 2], float* out) {
    float v[NV * VEC];
#pragma unroll
    for (int i = 0; i < NV * VEC / 2; ++i) {
        v[2 * i] = sum[i].x;
        v[2 * i + 1] = sum[i].y;
    }
    if (team.rows > 1) {
        __syncthreads();
        const int width = team.tpr * VEC * NV;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < VEC; ++i) shared[team.row * width + (j * team.tpr + team.me) * VEC + i] = v[j * VEC + i];
        __syncthreads();
        for (int c = threadIdx.x; c < p.channels; c += blockDim.x) {
            float s = 0.f;
            for (int r = 0; r < team.rows; ++r) s += shared[r * width + c];
            out[c] = s;
        }
        return;
    }
    constexpr int kPer = VEC < 4 ? VEC : 4;  // VEC divides the channels, so `out` starts on a vector
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = team.channel(j);
        if (!team.has(j)) continue;
#pragma unroll
        for (int i = 0; i < VEC; i += kPer) {
            Vec<float, kPer> o;
#pragma unroll
            for (int k = 0; k < kPer; ++k) o.w[k] = v[j * VEC + i + k];
            store_vec<float, kPer>(out, c + i, o);
        }
    }
}

// As kAhead: five tensors of 32 bytes per thread leave shared memory for one position.
template <int BYTES>
constexpr int kBackwardAhead = BYTES > 16 ? 1 : kAhead;

template <typename T, int VEC, int NV, int CL, int MODE>
__global__ void __launch_bounds__(kMaxThreads) token_backward_kernel(const __grid_constant__ Problem p, int tpr,
                                                                     int columns) {
    using F = Slots<T, VEC, NV>;
    constexpr int N = NV * VEC / 2, kTensors = backward_tensors(MODE), kDeep = kBackwardAhead<NV * sizeof(Vec<T, VEC>)>;
    // the tensors' places in a ring slot
    constexpr int kX = 0, kDn = 1, kDr = 2, kY = 3, kGate = 4;
    extern __shared__ __align__(16) unsigned char dynamic[];
    auto* part = reinterpret_cast<float*>(dynamic);
    grid_dep_launch();
    Team<VEC, CL> team(tpr, columns, p.channels, part);
    const int channels = p.channels;
    const long long block = blockIdx.x / CL;  // the cluster
    const F slots(dynamic + kPartBytes, team);
    const auto& on = slots.on;
    const long long first = tile_begin(p, block), last = tile_begin(p, block + 1);
    // a tile's sample and first position in it
    struct Cursor {
        long long sample, l;
        __device__ __forceinline__ void next(const Problem& p, int rows) {
            l += rows;
            if (l >= p.length) {
                l = 0;
                ++sample;
            }
        }
    };
    Cursor ahead = {first / p.tiles_per_sample, first % p.tiles_per_sample * team.rows};
    auto position = [&](const Cursor& c) { return c.sample * p.length + c.l + team.row; };
    auto here_at = [&](const Cursor& c) { return c.l + team.row < p.length; };
    auto row_at = [&](const Cursor& c) { return slots.row(static_cast<size_t>(position(c)) * channels, here_at(c)); };
    auto gate_at = [&](const Cursor& c) { return slots.row(static_cast<size_t>(c.sample) * channels, here_at(c)); };
    auto fetch = [&](long long tile, int ring) {
        if (tile < last) {
            const Row<NV> row = row_at(ahead);
            const unsigned k = ring * kTensors;
            if (p.dn) {
                slots.fetch(k + kX, p.x, row);
                slots.fetch(k + kDn, p.dn, row);
            }
            if (p.dr) slots.fetch(k + kDr, p.dr, row);
            if constexpr (MODE != kNoBlock) slots.fetch(k + kY, p.y, row);
            if constexpr (MODE == kFull) slots.fetch(k + kGate, p.gate, p.gate_mode == kGateSample ? gate_at(ahead) : row);
            ahead.next(p, team.rows);
        }
        copy_commit();
    };
    // the forward's statistics, a tile ahead too; zeros where there is no position
    auto saved = [&](const Cursor& c, bool exists) {
        return exists && here_at(c) ? reinterpret_cast<const float4*>(p.stats)[position(c)] : make_float4(0.f, 0.f, 0.f, 0.f);
    };
    Cursor now = ahead;
    float4 stats = saved(now, first < last);
#pragma unroll
    for (int k = 0; k < kDeep; ++k) fetch(first + k, k);
    const Weights<T, VEC, NV> weight_of(p, team, MODE != kNoBlock);
    float2 dw2[N], db2[N], tah[N], ta[N];
#pragma unroll
    for (int i = 0; i < N; ++i) dw2[i] = db2[i] = tah[i] = ta[i] = both(0.f);
    int turn = 0, ring = 0;
    for (long long tile = first; tile < last; ++tile) {
        const Row<NV> row = row_at(now);
        const bool here = here_at(now);
        const Row<NV> gate_row = p.gate_mode == kGateSample ? gate_at(now) : row;
        const long long sample = now.sample;
        const unsigned slot = ring * kTensors;
        const float2 rho = both(!p.post && here ? 1.f : p.post ? stats.y : 0.f);
        const float2 shift = both(p.post ? -stats.x * stats.y : 0.f);
        const float2 rho2 = both(p.dn ? stats.w : 0.f), shift2 = both(p.dn ? -stats.z * stats.w : 0.f);
        now.next(p, team.rows);
        stats = saved(now, tile + 1 < last);
        fetch(tile + kDeep, ring == 0 ? kDeep : ring - 1);
        copy_wait<kDeep>();
        // s: the sigmoid of the gate, or its plain value; the gate itself is read again where silu needs
        // it, since registers are what this kernel is short of
        float2 h[N], s[N], k[N], g[N];
        auto gate_of = [&](float2 (&a)[N]) {
#pragma unroll
            for (int i = 0; i < N; ++i) a[i] = s[i];
            if (p.act == kActSilu) {
                slots.read(slot + kGate, p.gate, gate_row, a);
#pragma unroll
                for (int i = 0; i < N; ++i) a[i] = mul2(a[i], s[i]);
            }
        };
        if constexpr (MODE != kNoBlock) {
            slots.read(slot + kY, p.y, row, h);
#pragma unroll
            for (int i = 0; i < N; ++i) h[i] = fma2(h[i], rho, shift);
            if constexpr (MODE == kFull) {
                slots.read(slot + kGate, p.gate, gate_row, s);
                if (p.act != kActNone) activate_all<T>(s, kActSigmoid);
            }
        }
        if (p.dn) {
            slots.read(slot + kX, p.x, row, k);
            slots.read(slot + kDn, p.dn, row, g);  // zeros where there is no channel
            float2 a[N];
            if constexpr (MODE == kFull) gate_of(a);
            float2 s0 = both(0.f), s1 = both(0.f);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                if constexpr (MODE != kNoBlock) {
                    const float2 z = fma2(h[i], weight_of.w[i], weight_of.b[i]);
                    k[i] = MODE == kPlain ? add2(k[i], z) : fma2(a[i], z, k[i]);
                }
                k[i] = fma2(k[i], rho2, shift2);
                dw2[i] = fma2(g[i], k[i], dw2[i]);
                db2[i] = add2(db2[i], g[i]);
                g[i] = mul2(g[i], weight_of.w2[i]);
                s0 = add2(s0, g[i]);
                s1 = fma2(g[i], k[i], s1);
            }
            float m[2] = {s0.x + s0.y, s1.x + s1.y};
            team.sum(m, turn);
            const float2 m1 = both(p.kind == kLayer ? -m[0] * p.inv_c : 0.f), m2 = both(-m[1] * p.inv_c);
#pragma unroll
            for (int i = 0; i < N; ++i) g[i] = mul2(rho2, add2(fma2(k[i], m2, g[i]), m1));
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) g[i] = both(0.f);
        }
        if (p.dr) {
            slots.read(slot + kDr, p.dr, row, k);
#pragma unroll
            for (int i = 0; i < N; ++i) g[i] = add2(g[i], k[i]);
        }
        clear_dead<VEC, NV>(g, on);
        // g: the gradient of r
        if (p.dx) slots.store(p.dx, row, g);
        if constexpr (MODE != kNoBlock) {
            float2 s0 = both(0.f), s1 = both(0.f), a[N];
            if constexpr (MODE == kFull) {
                gate_of(a);
                if (p.dgate && p.gate_mode == kGateFull) {
                    float2 o[N];
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        const float2 rest = make_float2(1.f - s[i].x, 1.f - s[i].y);
                        o[i] = p.act == kActSilu ? fma2(a[i], rest, s[i])
                                                 : p.act == kActSigmoid ? mul2(s[i], rest) : both(1.f);
                        o[i] = mul2(mul2(g[i], fma2(h[i], weight_of.w[i], weight_of.b[i])), o[i]);
                    }
                    slots.store(p.dgate, row, o);
                }
            }
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float2 v = MODE == kPlain ? g[i] : mul2(g[i], a[i]);
                const float2 kept = p.slots ? g[i] : v;
                tah[i] = fma2(kept, h[i], tah[i]);
                ta[i] = add2(ta[i], kept);
                k[i] = mul2(v, weight_of.w[i]);
                s0 = add2(s0, k[i]);
                s1 = fma2(k[i], h[i], s1);
            }
            if (p.dy) {
                if (p.post) {
                    float m[2] = {s0.x + s0.y, s1.x + s1.y};
                    team.sum(m, turn);
                    const float2 m3 = both(p.kind == kLayer ? -m[0] * p.inv_c : 0.f), m4 = both(-m[1] * p.inv_c);
#pragma unroll
                    for (int i = 0; i < N; ++i) k[i] = mul2(rho, add2(fma2(h[i], m4, k[i]), m3));
                }
                slots.store(p.dy, row, k);
            }
            if (p.slots && (tile + 1 == last || now.l == 0)) {
                // this ring slot has been read, and its next copies are kDeep positions away: the sums
                // of several rows meet in the space behind the ring
                float* meet = reinterpret_cast<float*>(dynamic + kPartBytes + (kDeep + 1) * kTensors * NV * slots.pitch);
                float* to = slot_of(p, block, sample);
                store_sums<VEC, NV>(p, team, meet, tah, to);
                store_sums<VEC, NV>(p, team, meet, ta, to + channels);
#pragma unroll
                for (int i = 0; i < N; ++i) tah[i] = ta[i] = both(0.f);
            }
        }
        ring = ring == kDeep ? 0 : ring + 1;
    }
    copy_wait<0>();
    if (!p.sums) return;
    float* meet = reinterpret_cast<float*>(dynamic + kPartBytes + (kDeep + 1) * kTensors * NV * slots.pitch);
    float* out = p.partial + static_cast<size_t>(block) * kSums * channels;
    store_sums<VEC, NV>(p, team, meet, dw2, out + static_cast<size_t>(kDPreW) * channels);
    store_sums<VEC, NV>(p, team, meet, db2, out + static_cast<size_t>(kDPreB) * channels);
    store_sums<VEC, NV>(p, team, meet, tah, out + static_cast<size_t>(kTah) * channels);
    store_sums<VEC, NV>(p, team, meet, ta, out + static_cast<size_t>(kTa) * channels);
}

// How a call's positions are laid over threads: tpr threads of each block of a cluster, `columns`
// channels of a block.
struct Lay {
    int tpr, columns, threads, rows;
    Lay(int channels, int vec, int nv, int cluster) {
        columns = ((channels + vec - 1) / vec + cluster - 1) / cluster * vec;
        tpr = 4;
        while (tpr * vec * nv < columns) tpr *= 2;
        threads = std::max(cluster > 1 ? kMaxThreads : 128, tpr);
        if (cluster > 1) tpr = kMaxThreads;
        rows = threads / tpr;
    }
};

template <int CL>
cudaError_t launch(const void* kernel, int clusters, int threads, size_t smem, cudaStream_t s, const Problem& p, Lay lay) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(clusters * CL);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim = {CL, 1, 1};
    cfg.attrs = attr;
    cfg.numAttrs = CL > 1 ? 1 : 0;
    Problem q = p;
    void* args[] = {&q, &lay.tpr, &lay.columns};
    return cudaLaunchKernelExC(&cfg, kernel, args);
}

template <typename T, int VEC, int NV, int CL, int MODE>
cudaError_t forward_as(const Problem& p, cudaStream_t s) {
    const Lay lay(p.channels, VEC, NV, CL);
    const long long groups = (p.positions + lay.rows - 1) / lay.rows;
    const size_t smem = kPartBytes + (kAhead + 1) * forward_tensors(MODE) * NV * sizeof(Vec<T, VEC>) * lay.threads;
    const void* kernel = reinterpret_cast<const void*>(token_forward_kernel<T, VEC, NV, CL, MODE>);
    int per_sm = 0;
    const cudaError_t e = scx::prepare_kernel(kernel, smem, lay.threads, &per_sm);
    if (e != cudaSuccess) return e;
    const int clusters = static_cast<int>(std::min<long long>(groups, std::max(1, per_sm * scx::num_sms() / CL)));
    return launch<CL>(kernel, clusters, lay.threads, smem, s, p, lay);
}

template <typename T, int VEC, int NV, int CL, int MODE>
cudaError_t backward_as(Problem& p, cudaStream_t s) {
    const Lay lay(p.channels, VEC, NV, CL);
    constexpr int kDeep = kBackwardAhead<NV * sizeof(Vec<T, VEC>)>;
    const size_t smem = kPartBytes + (kDeep + 1) * backward_tensors(MODE) * NV * sizeof(Vec<T, VEC>) * lay.threads +
                        (lay.rows > 1 ? sizeof(float) * lay.threads * VEC * NV : 0);
    const void* kernel = reinterpret_cast<const void*>(token_backward_kernel<T, VEC, NV, CL, MODE>);
    int per_sm = 0;
    const cudaError_t e = scx::prepare_kernel(kernel, smem, lay.threads, &per_sm);
    if (e != cudaSuccess) return e;
    p.tiles_per_sample = (p.length + lay.rows - 1) / lay.rows;
    p.tiles = p.batch * p.tiles_per_sample;
    p.parts = static_cast<int>(std::min<long long>(
        std::min(max_parts(p.channels), std::max(1, per_sm * scx::num_sms() / CL)), p.tiles));
    p.partials = p.parts;
    return launch<CL>(kernel, p.parts, lay.threads, smem, s, p, lay);
}

// Whether rows can be moved by vectors of VEC: whole ones per row, every base aligned, the weights for reads of
// VEC fp32 values (of four, where VEC is larger).
template <typename T, int VEC>
bool vectors_fit(const Problem& p) {
    const void* rows[] = {p.x, p.y, p.gate_mode != kGateNone ? p.gate : nullptr, p.r, p.n, p.dr, p.dn, p.dx, p.dy,
                          p.gate_mode == kGateFull ? p.dgate : nullptr};
    const void* weights[] = {p.post_w, p.post_b, p.pre_w, p.pre_b, p.scale_w};
    for (const void* a : rows)
        if (!aligned(a, VEC * sizeof(T))) return false;
    for (const void* a : weights)
        if (!aligned(a, std::min<size_t>(VEC, 4) * sizeof(float))) return false;
    return p.channels % VEC == 0;
}

// More per thread comes before a cluster: a position's sums within a block cost half of what a cluster's
// exchange does (4096 tokens of 8192 bf16 channels: forward 48 us, over two blocks 91).  What the forward keeps
// of 16 values fits its registers (all but 28 bytes in fp16 with a gate).  The backward's sums and weights do not: of 16 two-byte values it spills 416
// bytes without a gate, and is still the quicker there (training pass of the same tokens 195 us, over two blocks
// 217); with a gate it is not (304 and 265), and 8 values per thread are kept.
template <typename T, int MODE>
cudaError_t forward_in(const Problem& p, cudaStream_t s) {
    constexpr int VEC = 16 / static_cast<int>(sizeof(T));
    if (vectors_fit<T, VEC>(p)) {
        if (p.channels <= VEC * kMaxThreads) return forward_as<T, VEC, 1, 1, MODE>(p, s);
        if (p.channels <= 2 * VEC * kMaxThreads) return forward_as<T, VEC, 2, 1, MODE>(p, s);
        if (p.channels <= 4 * VEC * kMaxThreads) return forward_as<T, VEC, 2, 2, MODE>(p, s);
        return cudaErrorNotSupported;
    }
    if constexpr (sizeof(T) == 2)
        if (vectors_fit<T, 2>(p)) {
            if (p.channels <= 8 * kMaxThreads) return forward_as<T, 2, 4, 1, MODE>(p, s);
            if (p.channels <= 16 * kMaxThreads) return forward_as<T, 2, 4, 2, MODE>(p, s);
        }
    if (p.channels <= 4 * kMaxThreads) return forward_as<T, 1, 4, 1, MODE>(p, s);
    if (p.channels <= 8 * kMaxThreads) return forward_as<T, 1, 8, 1, MODE>(p, s);
    if (p.channels <= 16 * kMaxThreads) return forward_as<T, 1, 8, 2, MODE>(p, s);
    return cudaErrorNotSupported;
}

template <typename T, int MODE>
cudaError_t backward_in(Problem& p, cudaStream_t s) {
    constexpr int VEC = 16 / static_cast<int>(sizeof(T));
    if (vectors_fit<T, VEC>(p)) {
        if (p.channels <= VEC * kMaxThreads) return backward_as<T, VEC, 1, 1, MODE>(p, s);
        if constexpr (VEC == 4) {
            if (p.channels <= 8 * kMaxThreads) return backward_as<T, VEC, 2, 1, MODE>(p, s);
            if (p.channels <= 16 * kMaxThreads) return backward_as<T, VEC, 2, 2, MODE>(p, s);
        } else {
            if (p.channels <= 16 * kMaxThreads) {
                if constexpr (MODE == kFull) return backward_as<T, VEC, 1, 2, MODE>(p, s);
                else return backward_as<T, VEC, 2, 1, MODE>(p, s);
            }
            if (p.channels <= 32 * kMaxThreads) return backward_as<T, VEC, 1, 4, MODE>(p, s);
        }
        return cudaErrorNotSupported;
    }
    if constexpr (sizeof(T) == 2)
        if (vectors_fit<T, 2>(p)) {
            if (p.channels <= 8 * kMaxThreads) return backward_as<T, 2, 4, 1, MODE>(p, s);
            if (p.channels <= 16 * kMaxThreads) return backward_as<T, 2, 4, 2, MODE>(p, s);
        }
    if (p.channels <= 4 * kMaxThreads) return backward_as<T, 1, 4, 1, MODE>(p, s);
    if (p.channels <= 8 * kMaxThreads) return backward_as<T, 1, 8, 1, MODE>(p, s);
    if (p.channels <= 16 * kMaxThreads) return backward_as<T, 1, 8, 2, MODE>(p, s);
    return cudaErrorNotSupported;
}

}  // namespace

template <typename T>
cudaError_t token_forward(const Problem& p, cudaStream_t s) {
    switch (mode_of(p)) {
        case kNoBlock: return forward_in<T, kNoBlock>(p, s);
        case kPlain: return forward_in<T, kPlain>(p, s);
        default: return forward_in<T, kFull>(p, s);
    }
}

template <typename T>
cudaError_t token_backward(Problem& p, cudaStream_t s) {
    switch (mode_of(p)) {
        case kNoBlock: return backward_in<T, kNoBlock>(p, s);
        case kPlain: return backward_in<T, kPlain>(p, s);
        default: return backward_in<T, kFull>(p, s);
    }
}

}  // namespace scx_rn
