// block_gated.cu -- gated linear recurrence over long sequences, its gradient
// and its single steps.
//
//     h_t = f_t h_{t-1} + (1 - f_t) v_t,  f = 1 / (1 + e^-g)
//
// in terms of z = 1 - f alone: h += z (v - h).  f rounded to fp32 near 1
// would be off by a fixed 2^-25 in every step, which a memory of 1 / z steps
// multiplies; z is accurate to a few ulp however small it is.  Over a run of
// tokens the state goes from h to h - D h + B, where B is the run's answer
// from a zero state and D = 1 - prod(1 - z) its answer to v = 1 (the same
// recurrence), so D is as accurate as z.
//
// Bound by memory: every token is read once.  A CTA has 128 bytes of channels
// (4 per lane: 2 bf16 channels, worked on as a pair, or 1 f32) of one chunk of
// 128 tokens, a warp 8 consecutive tokens of it.  (D, B) of the warps meet in
// shared memory, those of the CTAs of a cluster (as many consecutive chunks of
// the same channels) in distributed shared memory; each CTA folds them onto
// the running state and the warps walk their tokens again.  Then the cluster
// moves on by its chunks.  The steps overlap: tiles arrive by TMA several
// steps ahead, and the gates and (D, B) of the next step are formed between
// arriving at the cluster's barrier and waiting for it.  Outputs overwrite
// their inputs' tile and leave by TMA.  Tensors that TMA cannot describe take
// the same kernel with plain loads, a lane's words one step ahead in its own
// slots of the tile, and plain stores.  Folds go in the order of the tokens:
// results do not depend on timing.
//
// The gradient walks the chunks from the end with c_t = f_t lam_t, the
// gradient that leaves token t for h_{t-1}: lam_t = dy_t + c_{t+1}, c_t =
// lam_t - z_t lam_t, so a run takes c to c - D c + E with the same D; h_{t-1}
// is walked forward again from the chunk's stored state.
//
// Sequences of up to 8 tokens (a decoder's step) need none of this: a warp
// walks its lanes' channels from global memory.
#include <cooperative_groups.h>

#include <cstring>

#include "block_common.cuh"
#include "common.cuh"
#include "tc_shared.cuh"

namespace hx {
namespace {

namespace cg = cooperative_groups;
using namespace umma;

constexpr int kChunk = HELIX_GATED_CHUNK;
constexpr int kTok = 8;                   // tokens of a warp
constexpr int kWarps = kChunk / kTok;
constexpr int kThreads = 32 * kWarps;
constexpr int kMaxCluster = 8;
constexpr int kTileBytes = kChunk * 128;  // 128 tokens x 128 bytes of channels
constexpr int kFewWarps = 8;              // of a CTA of the few-token kernels

// How a kernel reaches the token tensors.
enum Access { kTma, kWord, kHalf };       // tiles; a lane's 4 bytes; its 2-byte halves

// A lane's channels: one f32, or two bf16 as a packed fp32 pair.
template <typename T>
struct Lane;
template <>
struct Lane<float> {
    using V = float;
    static constexpr int kN = 1;
    static __device__ __forceinline__ V splat(float a) { return a; }
    static __device__ __forceinline__ V of(const float (&a)[1]) { return a[0]; }
    static __device__ __forceinline__ void to(V v, float (&a)[1]) { a[0] = v; }
    static __device__ __forceinline__ V fma(V a, V b, V c) { return fmaf(a, b, c); }
    static __device__ __forceinline__ V add(V a, V b) { return a + b; }
    static __device__ __forceinline__ V sub(V a, V b) { return a - b; }
    static __device__ __forceinline__ V mul(V a, V b) { return a * b; }
    static __device__ __forceinline__ V unpack(uint32_t w) { return __uint_as_float(w); }
    static __device__ __forceinline__ uint32_t pack(V v) { return __float_as_uint(v); }
    static constexpr uint32_t kInf = 0x7f800000u;
};
template <>
struct Lane<__nv_bfloat16> {
    using V = uint64_t;
    static constexpr int kN = 2;
    static __device__ __forceinline__ V splat(float a) { return f2_of(a, a); }
    static __device__ __forceinline__ V of(const float (&a)[2]) { return f2_of(a[0], a[1]); }
    static __device__ __forceinline__ void to(V v, float (&a)[2]) { f2_to(v, a[0], a[1]); }
    static __device__ __forceinline__ V fma(V a, V b, V c) { return f2_fma(a, b, c); }
    static __device__ __forceinline__ V add(V a, V b) { return f2_add(a, b); }
    static __device__ __forceinline__ V sub(V a, V b) { return f2_sub(a, b); }
    static __device__ __forceinline__ V mul(V a, V b) { return f2_mul(a, b); }
    static __device__ __forceinline__ V unpack(uint32_t w) { return f2_of_bf16x2(w); }
    static __device__ __forceinline__ uint32_t pack(V v) {
        float a[2];
        to(v, a);
        return bf16x2(a[0], a[1]);
    }
    static constexpr uint32_t kInf = 0x7f807f80u;
};

// z = 1 - sigmoid(g), accurate relative to z for every g down to subnormal z,
// and +infinity gives exactly 0 (what tokens past the end are given).
//
// z alone: with t = 2^-8 e^g, z = 2^-8 / (2^-8 + t).  The 2^-8 keeps the
// reciprocal's result normal until z is below 2^-134, so that small z come
// out as subnormals and not as zero.
template <typename T>
__device__ __forceinline__ typename Lane<T>::V gate(typename Lane<T>::V g) {
    using L = Lane<T>;
    float a[L::kN], r[L::kN];
    L::to(L::fma(g, L::splat(1.4426950408889634f), L::splat(-8.0f)), a);
#pragma unroll
    for (int e = 0; e < L::kN; ++e) asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(a[e]));
    L::to(L::add(L::of(a), L::splat(0x1p-8f)), r);
#pragma unroll
    for (int e = 0; e < L::kN; ++e) asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(r[e]));
    return L::mul(L::of(r), L::splat(0x1p-8f));
}
// With s = z (1 - z), which needs 1 - z just as accurate: t = e^-|g| (formed
// as 2^8 t, for the same reason), r = 1 / (1 + t), sigmoid(|g|) = r,
// sigmoid(-|g|) = t r.
template <typename T>
__device__ __forceinline__ void gate_slope(typename Lane<T>::V g, typename Lane<T>::V& z, typename Lane<T>::V& s) {
    using L = Lane<T>;
    float x[L::kN], t[L::kN], r[L::kN], zz[L::kN];
    L::to(g, x);
#pragma unroll
    for (int e = 0; e < L::kN; ++e) {
        t[e] = fmaf(-fabsf(x[e]), 1.4426950408889634f, 8.0f);
        asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(t[e]));
    }
    const typename L::V tv = L::mul(L::of(t), L::splat(0x1p-8f));
    L::to(L::add(tv, L::splat(1.0f)), r);
#pragma unroll
    for (int e = 0; e < L::kN; ++e) asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(r[e]));
    const typename L::V tr = L::mul(tv, L::of(r));
    L::to(tr, t);
#pragma unroll
    for (int e = 0; e < L::kN; ++e) zz[e] = x[e] >= 0.0f ? t[e] : r[e];
    z = L::of(zz);
    s = L::mul(tr, L::of(r));
}

// h - d h + b
template <typename L>
__device__ __forceinline__ typename L::V fold(typename L::V h, typename L::V d, typename L::V b) {
    return L::add(L::sub(h, L::mul(d, h)), b);
}
// a + z (v - a): a step of the recurrence, and (v = 1) of D
template <typename L>
__device__ __forceinline__ typename L::V step(typename L::V a, typename L::V z, typename L::V v) {
    return L::fma(z, L::sub(v, a), a);
}

// A lane's 4 bytes of a row; n: its channels that exist.
template <typename T, Access A>
__device__ __forceinline__ uint32_t ld_raw(const T* p, int n) {
    if (sizeof(T) == 4 || (A != kHalf && n == 2)) return __ldcs(reinterpret_cast<const unsigned int*>(p));
    const unsigned short* q = reinterpret_cast<const unsigned short*>(p);
    const uint32_t lo = __ldcs(q), up = n == 2 ? __ldcs(q + 1) : 0;
    return lo | up << 16;
}
template <typename T, Access A>
__device__ __forceinline__ void st_raw(T* p, int n, uint32_t w) {
    if (sizeof(T) == 4 || (A != kHalf && n == 2)) {
        __stcs(reinterpret_cast<unsigned int*>(p), w);
        return;
    }
    unsigned short* q = reinterpret_cast<unsigned short*>(p);
    q[0] = (unsigned short)w;
    if (n == 2) q[1] = (unsigned short)(w >> 16);
}
template <typename L>
__device__ __forceinline__ typename L::V ld_state(const float* p, int n) {
    float a[L::kN];
#pragma unroll
    for (int e = 0; e < L::kN; ++e) a[e] = p && e < n ? p[e] : 0.0f;
    return L::of(a);
}
template <typename L>
__device__ __forceinline__ void st_state(float* p, int n, typename L::V v) {
    float a[L::kN];
    L::to(v, a);
#pragma unroll
    for (int e = 0; e < L::kN; ++e)
        if (e < n) p[e] = a[e];
}

__device__ __forceinline__ int length_of(const GatedParams& p, int seq) {
    return p.lengths ? min(max(p.lengths[seq], 0), p.n_tok) : p.n_tok;
}

// Where a thread is: its group of channels, and its tokens of a chunk.
template <typename T>
struct Place {
    int warp, lane, rank, seq, c0, n, len;
    __device__ __forceinline__ Place(const GatedParams& p) {
        constexpr int N = Lane<T>::kN, CB = 32 * N;
        warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0);
        lane = threadIdx.x & 31;
        rank = (int)(blockIdx.x % (unsigned)p.cluster);
        const int slabs = (p.n_chan + CB - 1) / CB;
        const unsigned group = blockIdx.x / (unsigned)p.cluster;
        seq = (int)(group / (unsigned)slabs);
        c0 = (int)(group % (unsigned)slabs) * CB + N * lane;
        n = max(0, min(N, p.n_chan - c0));
        len = length_of(p, seq);
    }
    __device__ __forceinline__ int slab0() const { return c0 - Lane<T>::kN * lane; }
};

// The warps' (D, B) of a step, and the totals of the cluster's CTAs; two
// steps' worth each, since a warp may be a step ahead of another.
template <typename V, int K>
struct Meet {
    V warp[2][K][kWarps][32];
    V total[2][2][kMaxCluster][32];
};

__device__ __forceinline__ void cluster_arrive() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void bulk_wait_read() {
    asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}

struct GatedMaps {
    CUtensorMap in[3], out[2];  // g, v, dy; y, or dg and dv
};

// The tiles of the steps to come: K input tensors per stage.
template <typename T, Access A, int K, int kStages>
struct Tiles {
    uint8_t*  base;
    uint64_t* full;
    bool      alive = true;

    __device__ __forceinline__ uint8_t* tile(int turn, int k) const {
        return base + ((turn % kStages) * K + k) * kTileBytes;
    }
    __device__ __forceinline__ uint32_t* word(int turn, int k, int row, int lane) const {
        return reinterpret_cast<uint32_t*>(tile(turn, k) + row * 128 + lane * 4);
    }
    // One thread: turn's tiles start to arrive.
    __device__ __forceinline__ void load(const GatedMaps& m, int turn, int c0, int t0, int seq) const {
        uint64_t* bar = &full[turn % kStages];
        mbar_expect_tx(bar, K * kTileBytes);
#pragma unroll
        for (int k = 0; k < K; ++k) tma_load_3d(tile(turn, k), &m.in[k], bar, c0, t0, seq);
    }
    __device__ __forceinline__ void wait(int turn, unsigned* fault) {
        if (A != kTma || !alive) return;
        alive = mbar_wait(&full[turn % kStages], (uint32_t)((turn / kStages) & 1), tc::kWaitBudget);
        if (!alive && fault) atomicCAS(fault, 0u, (unsigned)kFaultGated);
        __syncwarp();
    }
};

template <typename T, Access A, int kStages>
__global__ void __launch_bounds__(kThreads, 1)
    gated_kernel(const __grid_constant__ GatedMaps maps, const GatedParams p) {
    using L = Lane<T>;
    using V = typename L::V;
    extern __shared__ uint8_t smem_raw[];
    __shared__ Meet<V, 2> meet;
    __shared__ uint64_t full[kStages];
    cg::cluster_group cluster = cg::this_cluster();

    const Place<T> at(p);
    const int R = p.cluster, steps = (p.n_chunk + R - 1) / R;
    const int warp = at.warp, lane = at.lane, n = at.n;
    const bool issuer = threadIdx.x == kThreads - 1;
    Tiles<T, A, 2, kStages> tiles{reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 127) & ~uintptr_t(127)),
                                  full};

    const T* src[2] = {static_cast<const T*>(p.g) + (int64_t)at.seq * p.seq_g + at.c0,
                       static_cast<const T*>(p.v) + (int64_t)at.seq * p.seq_v + at.c0};
    const int64_t pitch[2] = {p.s_g, p.s_v};
    T* y = static_cast<T*>(p.y) + (int64_t)at.seq * p.seq_y + at.c0;

    auto chunk_of = [&](int s) { return s * R + at.rank; };
    uint32_t ahead[A == kTma ? 1 : 2][A == kTma ? 1 : kTok];
    auto fetch = [&](int s) {  // plain access: the lane's words of step s
        if constexpr (A != kTma) {
            const int t0 = chunk_of(s) * kChunk + warp * kTok;
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int i = 0; i < kTok; ++i)
                    ahead[k][i] = n > 0 && t0 + i < at.len ? ld_raw<T, A>(src[k] + (t0 + i) * pitch[k], n) : 0u;
        }
    };
    auto keep = [&](int s) {
        if constexpr (A != kTma) {
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int i = 0; i < kTok; ++i) *tiles.word(s, k, warp * kTok + i, lane) = ahead[k][i];
        }
    };

    if (A == kTma) {
        if (issuer) {
#pragma unroll
            for (int k = 0; k < kStages; ++k) mbar_init(&full[k], 1);
            fence_mbar_init();
            for (int s = 0; s < kStages && s < steps; ++s)
                tiles.load(maps, s, at.slab0(), chunk_of(s) * kChunk, at.seq);
        }
        __syncthreads();
    }

    V h = ld_state<L>(p.h0 ? p.h0 + (int64_t)at.seq * p.seq_h0 + at.c0 : nullptr, n);
    V z[kTok], zn[kTok], D, B;
    // gates and the warp's (D, B) of step s
    auto first = [&](int s, V(&zs)[kTok]) {
        tiles.wait(s, p.fault);
        const int t0 = chunk_of(s) * kChunk + warp * kTok;
        const bool whole = t0 + kTok <= at.len;
        D = B = L::splat(0.0f);
#pragma unroll
        for (int i = 0; i < kTok; ++i) {
            uint32_t gw = *tiles.word(s, 0, warp * kTok + i, lane), vw = *tiles.word(s, 1, warp * kTok + i, lane);
            if (!whole && t0 + i >= at.len) gw = L::kInf, vw = 0u;
            zs[i] = gate<T>(L::unpack(gw));
            D = step<L>(D, zs[i], L::splat(1.0f));
            B = step<L>(B, zs[i], L::unpack(vw));
        }
    };
    // shares them: within the CTA, then its totals with the cluster
    auto publish = [&](int s) {
        const int b = s & 1;
        meet.warp[b][0][warp][lane] = D;
        meet.warp[b][1][warp][lane] = B;
        __syncthreads();
        if (warp < R) {
            V d = L::splat(0.0f), t = d;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const V dw = meet.warp[b][0][w][lane];
                d = step<L>(d, dw, L::splat(1.0f));
                t = fold<L>(t, dw, meet.warp[b][1][w][lane]);
            }
            Meet<V, 2>* to = cluster.map_shared_rank(&meet, warp);
            to->total[b][0][at.rank][lane] = d;
            to->total[b][1][at.rank][lane] = t;
        }
        cluster_arrive();
    };

    // no CTA writes to another's shared memory before that one runs
    cluster_arrive();
    cluster_wait();
    if (steps > 0) {
        fetch(0);
        keep(0);
        if (steps > 1) {
            fetch(1);
            keep(1);
        }
        first(0, z);
        publish(0);
    }
    for (int s = 0; s < steps; ++s) {
        const int chunk = chunk_of(s), b = s & 1, t0 = chunk * kChunk + warp * kTok;
        if (s + 2 < steps) fetch(s + 2);
        if (s + 1 < steps) first(s + 1, zn);
        cluster_wait();
        V hw = h;
        for (int k = 0; k < R; ++k) {
            if (k == at.rank) hw = h;
            h = fold<L>(h, meet.total[b][0][k][lane], meet.total[b][1][k][lane]);
        }
        if (p.states && warp == 0 && chunk < p.n_chunk)
            st_state<L>(p.states + ((int64_t)at.seq * p.n_chunk + chunk) * p.n_chan + at.c0, n, hw);
        for (int w = 0; w < warp; ++w)
            hw = fold<L>(hw, meet.warp[b][0][w][lane], meet.warp[b][1][w][lane]);
        const bool whole = t0 + kTok <= at.len;
#pragma unroll
        for (int i = 0; i < kTok; ++i) {
            uint32_t* slot = tiles.word(s, 1, warp * kTok + i, lane);
            const bool past = !whole && t0 + i >= at.len;
            hw = step<L>(hw, z[i], past ? L::splat(0.0f) : L::unpack(*slot));
            const uint32_t o = past ? 0u : L::pack(hw);
            if (A == kTma)
                *slot = o;
            else if (t0 + i < p.n_tok && n > 0)
                st_raw<T, A>(y + (t0 + i) * p.s_y, n, o);
        }
        if (s + 2 < steps) keep(s + 2);
        if (A == kTma) fence_async_smem();
        if (s + 1 < steps)
            publish(s + 1);
        else
            __syncthreads();
        if (A == kTma && issuer) {
            if (chunk < p.n_chunk) tma_store_3d(&maps.out[0], tiles.tile(s, 1), at.slab0(), chunk * kChunk, at.seq);
            bulk_commit();
            // the stage of the step before is free once its output has been read
            if (s >= 1 && s - 1 + kStages < steps) {
                bulk_wait_read<1>();
                tiles.load(maps, s - 1 + kStages, at.slab0(), chunk_of(s - 1 + kStages) * kChunk, at.seq);
            }
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < kTok; ++i) z[i] = zn[i];
    }
    if (A == kTma && issuer) {
        // whatever the other threads made of their waits, the loads land
        for (int s = max(0, steps - kStages); s < steps; ++s)
            mbar_wait(&full[s % kStages], (uint32_t)((s / kStages) & 1), tc::kWaitBudget);
        bulk_wait0();
    }
    // Every CTA holds the last state.  In place of h0 is safe: each has read
    // h0 before the cluster's first barrier.
    if (at.rank == 0 && warp == 0) st_state<L>(p.h1 + (int64_t)at.seq * p.seq_h1 + at.c0, n, h);
}

template <typename T, Access A, int kStages>
__global__ void __launch_bounds__(kThreads, 1)
    gated_grad_kernel(const __grid_constant__ GatedMaps maps, const GatedParams p) {
    using L = Lane<T>;
    using V = typename L::V;
    extern __shared__ uint8_t smem_raw[];
    __shared__ Meet<V, 3> meet;
    __shared__ uint64_t full[kStages];
    cg::cluster_group cluster = cg::this_cluster();

    const Place<T> at(p);
    const int R = p.cluster, steps = (p.n_chunk + R - 1) / R;
    const int warp = at.warp, lane = at.lane, n = at.n;
    const bool issuer = threadIdx.x == kThreads - 1;
    Tiles<T, A, 3, kStages> tiles{reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 127) & ~uintptr_t(127)),
                                  full};

    const T* src[3] = {static_cast<const T*>(p.g) + (int64_t)at.seq * p.seq_g + at.c0,
                       static_cast<const T*>(p.v) + (int64_t)at.seq * p.seq_v + at.c0,
                       static_cast<const T*>(p.dy) + (int64_t)at.seq * p.seq_dy + at.c0};
    const int64_t pitch[3] = {p.s_g, p.s_v, p.s_dy};
    T* dg = static_cast<T*>(p.dg) + (int64_t)at.seq * p.seq_dg + at.c0;
    T* dv = static_cast<T*>(p.dv) + (int64_t)at.seq * p.seq_dv + at.c0;

    // turns count from the end
    auto chunk_of = [&](int s) { return (steps - 1 - s) * R + at.rank; };
    uint32_t ahead[A == kTma ? 1 : 3][A == kTma ? 1 : kTok];
    auto fetch = [&](int s) {
        if constexpr (A != kTma) {
            const int t0 = chunk_of(s) * kChunk + warp * kTok;
#pragma unroll
            for (int k = 0; k < 3; ++k)
#pragma unroll
                for (int i = 0; i < kTok; ++i)
                    ahead[k][i] = n > 0 && t0 + i < at.len ? ld_raw<T, A>(src[k] + (t0 + i) * pitch[k], n) : 0u;
        }
    };
    auto keep = [&](int s) {
        if constexpr (A != kTma) {
#pragma unroll
            for (int k = 0; k < 3; ++k)
#pragma unroll
                for (int i = 0; i < kTok; ++i) *tiles.word(s, k, warp * kTok + i, lane) = ahead[k][i];
        }
    };

    if (A == kTma) {
        if (issuer) {
#pragma unroll
            for (int k = 0; k < kStages; ++k) mbar_init(&full[k], 1);
            fence_mbar_init();
            for (int s = 0; s < kStages && s < steps; ++s)
                tiles.load(maps, s, at.slab0(), chunk_of(s) * kChunk, at.seq);
        }
        __syncthreads();
    }

    V c = ld_state<L>(p.dh1 ? p.dh1 + (int64_t)at.seq * p.seq_dh1 + at.c0 : nullptr, n);
    V z[kTok], q[kTok], zn[kTok], qn[kTok], D, B, E, h, hn;
    auto first = [&](int s, V(&zs)[kTok], V(&qs)[kTok], V& hs) {
        const int chunk = chunk_of(s), t0 = chunk * kChunk + warp * kTok;
        hs = ld_state<L>(chunk < p.n_chunk ? p.states + ((int64_t)at.seq * p.n_chunk + chunk) * p.n_chan + at.c0 : nullptr,
                         n);
        tiles.wait(s, p.fault);
        const bool whole = t0 + kTok <= at.len;
        D = B = E = L::splat(0.0f);
#pragma unroll
        for (int i = 0; i < kTok; ++i) {
            uint32_t gw = *tiles.word(s, 0, warp * kTok + i, lane), vw = *tiles.word(s, 1, warp * kTok + i, lane);
            if (!whole && t0 + i >= at.len) gw = L::kInf, vw = 0u;
            gate_slope<T>(L::unpack(gw), zs[i], qs[i]);
            D = step<L>(D, zs[i], L::splat(1.0f));
            B = step<L>(B, zs[i], L::unpack(vw));
        }
#pragma unroll
        for (int i = kTok - 1; i >= 0; --i) {
            uint32_t yw = *tiles.word(s, 2, warp * kTok + i, lane);
            if (!whole && t0 + i >= at.len) yw = 0u;
            const V lam = L::add(L::unpack(yw), E);
            E = L::sub(lam, L::mul(zs[i], lam));
        }
    };
    auto publish = [&](int s) {
        const int b = s & 1;
        meet.warp[b][0][warp][lane] = D;
        meet.warp[b][1][warp][lane] = B;
        meet.warp[b][2][warp][lane] = E;
        __syncthreads();
        if (warp < R) {
            V d = L::splat(0.0f), t = d;
#pragma unroll
            for (int w = kWarps - 1; w >= 0; --w) {
                const V dw = meet.warp[b][0][w][lane];
                d = step<L>(d, dw, L::splat(1.0f));
                t = fold<L>(t, dw, meet.warp[b][2][w][lane]);
            }
            Meet<V, 3>* to = cluster.map_shared_rank(&meet, warp);
            to->total[b][0][at.rank][lane] = d;
            to->total[b][1][at.rank][lane] = t;
        }
        cluster_arrive();
    };

    cluster_arrive();
    cluster_wait();
    if (steps > 0) {
        fetch(0);
        keep(0);
        if (steps > 1) {
            fetch(1);
            keep(1);
        }
        first(0, z, q, h);
        publish(0);
    }
    for (int s = 0; s < steps; ++s) {
        const int chunk = chunk_of(s), b = s & 1, t0 = chunk * kChunk + warp * kTok;
        const bool whole = t0 + kTok <= at.len;
        if (s + 2 < steps) fetch(s + 2);
        // h_{t-1} - v_t of the warp's tokens
        for (int w = 0; w < warp; ++w)
            h = fold<L>(h, meet.warp[b][0][w][lane], meet.warp[b][1][w][lane]);
#pragma unroll
        for (int i = 0; i < kTok; ++i) {
            uint32_t vw = *tiles.word(s, 1, warp * kTok + i, lane);
            if (!whole && t0 + i >= at.len) vw = 0u;
            const V off = L::sub(h, L::unpack(vw));
            q[i] = L::mul(q[i], off);
            h = L::sub(h, L::mul(z[i], off));
        }
        if (s + 1 < steps) first(s + 1, zn, qn, hn);
        cluster_wait();
        V cw = c;
        for (int k = R - 1; k >= 0; --k) {
            if (k == at.rank) cw = c;
            c = fold<L>(c, meet.total[b][0][k][lane], meet.total[b][1][k][lane]);
        }
        for (int w = kWarps - 1; w > warp; --w)
            cw = fold<L>(cw, meet.warp[b][0][w][lane], meet.warp[b][2][w][lane]);
#pragma unroll
        for (int i = kTok - 1; i >= 0; --i) {
            const int row = warp * kTok + i;
            const bool past = !whole && t0 + i >= at.len;
            const V lam = L::add(past ? L::splat(0.0f) : L::unpack(*tiles.word(s, 2, row, lane)), cw);
            const V zl = L::mul(z[i], lam);
            const uint32_t og = past ? 0u : L::pack(L::mul(lam, q[i])), ov = past ? 0u : L::pack(zl);
            cw = L::sub(lam, zl);
            if (A == kTma) {
                *tiles.word(s, 0, row, lane) = og;
                *tiles.word(s, 1, row, lane) = ov;
            } else if (t0 + i < p.n_tok && n > 0) {
                st_raw<T, A>(dg + (t0 + i) * p.s_dg, n, og);
                st_raw<T, A>(dv + (t0 + i) * p.s_dv, n, ov);
            }
        }
        if (s + 2 < steps) keep(s + 2);
        if (A == kTma) fence_async_smem();
        if (s + 1 < steps)
            publish(s + 1);
        else
            __syncthreads();
        if (A == kTma && issuer) {
            if (chunk < p.n_chunk) {
                tma_store_3d(&maps.out[0], tiles.tile(s, 0), at.slab0(), chunk * kChunk, at.seq);
                tma_store_3d(&maps.out[1], tiles.tile(s, 1), at.slab0(), chunk * kChunk, at.seq);
            }
            bulk_commit();
            if (s >= 1 && s - 1 + kStages < steps) {
                bulk_wait_read<1>();
                tiles.load(maps, s - 1 + kStages, at.slab0(), chunk_of(s - 1 + kStages) * kChunk, at.seq);
            }
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < kTok; ++i) z[i] = zn[i], q[i] = qn[i];
        h = hn;
    }
    if (A == kTma && issuer) {
        for (int s = max(0, steps - kStages); s < steps; ++s)
            mbar_wait(&full[s % kStages], (uint32_t)((s / kStages) & 1), tc::kWaitBudget);
        bulk_wait0();
    }
    if (p.dh0 && at.rank == 0 && warp == 0) st_state<L>(p.dh0 + (int64_t)at.seq * p.seq_dh0 + at.c0, n, c);
}

// Up to kTok tokens: a warp has the channels of one slab of one sequence.
template <typename T, Access A, bool GRAD>
__global__ void __launch_bounds__(32 * kFewWarps) gated_few_kernel(const GatedParams p) {
    using L = Lane<T>;
    using V = typename L::V;
    constexpr int N = L::kN, CB = 32 * N;
    const int slabs = (p.n_chan + CB - 1) / CB;
    const int64_t group = (int64_t)blockIdx.x * kFewWarps + (threadIdx.x >> 5);
    if (group >= (int64_t)p.n_seq * slabs) return;
    const int seq = (int)(group / slabs), c0 = (int)(group % slabs) * CB + N * (int)(threadIdx.x & 31);
    const int n = min(N, p.n_chan - c0);
    if (n <= 0) return;
    const int len = length_of(p, seq);
    const T* g = static_cast<const T*>(p.g) + (int64_t)seq * p.seq_g + c0;
    const T* v = static_cast<const T*>(p.v) + (int64_t)seq * p.seq_v + c0;
    const T* dy = static_cast<const T*>(p.dy) + (int64_t)seq * p.seq_dy + c0;

    V z[kTok], q[GRAD ? kTok : 1];
    uint32_t vw[kTok], yw[GRAD ? kTok : 1];
#pragma unroll
    for (int i = 0; i < kTok; ++i) {
        const bool live = i < len;
        const uint32_t gw = live ? ld_raw<T, A>(g + i * p.s_g, n) : L::kInf;
        vw[i] = live ? ld_raw<T, A>(v + i * p.s_v, n) : 0u;
        if constexpr (GRAD) yw[i] = live ? ld_raw<T, A>(dy + i * p.s_dy, n) : 0u;
        if constexpr (GRAD)
            gate_slope<T>(L::unpack(gw), z[i], q[i]);
        else
            z[i] = gate<T>(L::unpack(gw));
    }
    if constexpr (!GRAD) {
        T* y = static_cast<T*>(p.y) + (int64_t)seq * p.seq_y + c0;
        V h = ld_state<L>(p.h0 ? p.h0 + (int64_t)seq * p.seq_h0 + c0 : nullptr, n);
        if (p.states && p.n_tok > 0) st_state<L>(p.states + (int64_t)seq * p.n_chan + c0, n, h);
#pragma unroll
        for (int i = 0; i < kTok; ++i) {
            if (i < len) h = step<L>(h, z[i], L::unpack(vw[i]));
            if (i < p.n_tok) st_raw<T, A>(y + i * p.s_y, n, i < len ? L::pack(h) : 0u);
        }
        st_state<L>(p.h1 + (int64_t)seq * p.seq_h1 + c0, n, h);
    } else {
        T* dg = static_cast<T*>(p.dg) + (int64_t)seq * p.seq_dg + c0;
        T* dv = static_cast<T*>(p.dv) + (int64_t)seq * p.seq_dv + c0;
        V h = ld_state<L>(p.n_tok > 0 ? p.states + (int64_t)seq * p.n_chan + c0 : nullptr, n);
#pragma unroll
        for (int i = 0; i < kTok; ++i) {
            const V off = L::sub(h, L::unpack(vw[i]));
            q[i] = L::mul(q[i], off);
            h = L::sub(h, L::mul(z[i], off));
        }
        V c = ld_state<L>(p.dh1 ? p.dh1 + (int64_t)seq * p.seq_dh1 + c0 : nullptr, n);
#pragma unroll
        for (int i = kTok - 1; i >= 0; --i) {
            if (i >= p.n_tok) continue;
            const bool live = i < len;
            const V lam = L::add(L::unpack(yw[i]), c), zl = L::mul(z[i], lam);
            st_raw<T, A>(dg + i * p.s_dg, n, live ? L::pack(L::mul(lam, q[i])) : 0u);
            st_raw<T, A>(dv + i * p.s_dv, n, live ? L::pack(zl) : 0u);
            if (live) c = L::sub(lam, zl);
        }
        if (p.dh0) st_state<L>(p.dh0 + (int64_t)seq * p.seq_dh0 + c0, n, c);
    }
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------
// One CTA per SM.  At the end of a step the tiles of that step and the next
// are still held: the loads run kStages - 2 steps ahead of their use.
constexpr int kFwdStages = 6, kGradStages = 4;
constexpr size_t kFwdSmem = (size_t)kFwdStages * 2 * kTileBytes + 128;
constexpr size_t kGradSmem = (size_t)kGradStages * 3 * kTileBytes + 128;

// [n_seq][n_tok][n_chan] in boxes of 128 tokens x 128 bytes; false when TMA
// cannot describe it.  Rows and channels past the ends read as zero and are
// not written.
bool make_map_tok(const helix_ctx* ctx, CUtensorMap* m, const GatedParams& p, const void* base, int64_t s_tok,
                  int64_t s_seq, int size) {
    if (reinterpret_cast<uintptr_t>(base) % 16) return false;
    const int64_t row = ((int64_t)p.n_chan * size + 15) / 16 * 16;
    const int64_t bt = p.n_tok > 1 ? s_tok * size : row, bs = p.n_seq > 1 ? s_seq * size : row;
    if (bt <= 0 || bs <= 0 || bt % 16 || bs % 16) return false;
    const auto fn = reinterpret_cast<tc::EncodeFn>(ctx->encode_tiled);
    cuuint64_t dims[3] = {(cuuint64_t)p.n_chan, (cuuint64_t)p.n_tok, (cuuint64_t)p.n_seq};
    cuuint64_t strides[2] = {(cuuint64_t)bt, (cuuint64_t)bs};
    cuuint32_t box[3] = {(cuuint32_t)(128 / size), (cuuint32_t)kChunk, 1};
    cuuint32_t es[3] = {1, 1, 1};
    return fn(m, size == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
              const_cast<void*>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool make_maps(const helix_ctx* ctx, GatedMaps* m, const GatedParams& p, bool grad, int size) {
    std::memset(m, 0, sizeof(*m));
    if (!ctx->encode_tiled || p.n_tok <= 0) return false;
    if (!make_map_tok(ctx, &m->in[0], p, p.g, p.s_g, p.seq_g, size)) return false;
    if (!make_map_tok(ctx, &m->in[1], p, p.v, p.s_v, p.seq_v, size)) return false;
    if (!grad) return make_map_tok(ctx, &m->out[0], p, p.y, p.s_y, p.seq_y, size);
    return make_map_tok(ctx, &m->in[2], p, p.dy, p.s_dy, p.seq_dy, size) &&
           make_map_tok(ctx, &m->out[0], p, p.dg, p.s_dg, p.seq_dg, size) &&
           make_map_tok(ctx, &m->out[1], p, p.dv, p.s_dv, p.seq_dv, size);
}

// CTAs of a cluster: the size with the fewest steps, counting the waves that
// its clusters take, one CTA per SM (large clusters leave SMs of a GPC idle),
// and two steps to fill and drain each.
int cluster_of(const helix_ctx* ctx, int64_t groups, int chunks) {
    int best = 1;
    int64_t least = INT64_MAX;
    for (int i = 0, r = 1; r <= kMaxCluster; ++i, r *= 2) {
        const int64_t at_once = ctx->gated_clusters[i];
        if (at_once <= 0 || (r > 1 && r >= 2 * chunks)) continue;
        const int64_t cost = (groups + at_once - 1) / at_once * ((chunks + r - 1) / r + 2);
        if (cost < least) least = cost, best = r;
    }
    return best;
}

template <typename T, Access A>
int launch_gated_a(const helix_ctx* ctx, const GatedMaps& maps, GatedParams p, bool grad, void* stream) {
    constexpr int CB = 32 * Lane<T>::kN;
    constexpr Access few = A == kTma ? kWord : A;
    const int64_t groups = (int64_t)p.n_seq * ((p.n_chan + CB - 1) / CB);
    if (p.n_tok <= kTok) {
        const dim3 grid((unsigned)((groups + kFewWarps - 1) / kFewWarps)), block(32 * kFewWarps);
        return grad ? block_launch(gated_few_kernel<T, few, true>, grid, block, 0, stream, p)
                    : block_launch(gated_few_kernel<T, few, false>, grid, block, 0, stream, p);
    }
    p.cluster = cluster_of(ctx, groups, p.n_chunk);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(groups * p.cluster));
    cfg.blockDim = dim3((unsigned)kThreads);
    cfg.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = (unsigned)p.cluster;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    cfg.dynamicSmemBytes = grad ? kGradSmem : kFwdSmem;
    return grad ? cudaLaunchKernelEx(&cfg, gated_grad_kernel<T, A, kGradStages>, maps, p)
                : cudaLaunchKernelEx(&cfg, gated_kernel<T, A, kFwdStages>, maps, p);
}

int launch_gated_any(const helix_ctx* ctx, const helix_gated_scan_desc& d, const GatedParams& p, bool word, bool grad,
                     void* stream) {
    GatedMaps maps;
    const bool tma = p.n_tok > kTok && make_maps(ctx, &maps, p, grad, d.io_dtype == HELIX_F32 ? 4 : 2);
    if (d.io_dtype == HELIX_F32)
        return tma ? launch_gated_a<float, kTma>(ctx, maps, p, grad, stream)
                   : launch_gated_a<float, kWord>(ctx, maps, p, grad, stream);
    if (tma) return launch_gated_a<__nv_bfloat16, kTma>(ctx, maps, p, grad, stream);
    return word ? launch_gated_a<__nv_bfloat16, kWord>(ctx, maps, p, grad, stream)
                : launch_gated_a<__nv_bfloat16, kHalf>(ctx, maps, p, grad, stream);
}

template <typename T, Access A>
int configure_gated_a() {
    const int e = cudaFuncSetAttribute(gated_kernel<T, A, kFwdStages>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       (int)kFwdSmem);
    if (e != cudaSuccess) return e;
    return cudaFuncSetAttribute(gated_grad_kernel<T, A, kGradStages>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                (int)kGradSmem);
}

}  // namespace

int configure_gated(helix_ctx* ctx) {
    int e;
    if ((e = configure_gated_a<float, kTma>()) != cudaSuccess) return e;
    if ((e = configure_gated_a<float, kWord>()) != cudaSuccess) return e;
    if ((e = configure_gated_a<__nv_bfloat16, kTma>()) != cudaSuccess) return e;
    if ((e = configure_gated_a<__nv_bfloat16, kWord>()) != cudaSuccess) return e;
    if ((e = configure_gated_a<__nv_bfloat16, kHalf>()) != cudaSuccess) return e;
    for (int i = 0, r = 1; r <= kMaxCluster; ++i, r *= 2) {
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3((unsigned)r);
        cfg.blockDim = dim3((unsigned)kThreads);
        cfg.dynamicSmemBytes = kFwdSmem;
        cudaLaunchAttribute at{};
        at.id = cudaLaunchAttributeClusterDimension;
        at.val.clusterDim.x = (unsigned)r;
        at.val.clusterDim.y = at.val.clusterDim.z = 1;
        cfg.attrs = &at;
        cfg.numAttrs = 1;
        e = cudaOccupancyMaxActiveClusters(&ctx->gated_clusters[i], gated_kernel<__nv_bfloat16, kTma, kFwdStages>, &cfg);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

int launch_gated(const helix_ctx* ctx, const helix_gated_scan_desc& d, GatedParams p, bool word, void* stream) {
    return launch_gated_any(ctx, d, p, word, false, stream);
}

int launch_gated_grad(const helix_ctx* ctx, const helix_gated_scan_desc& d, GatedParams p, bool word, void* stream) {
    return launch_gated_any(ctx, d, p, word, true, stream);
}

}  // namespace hx
