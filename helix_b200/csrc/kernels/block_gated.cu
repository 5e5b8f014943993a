// block_gated.cu -- gated linear recurrence over long sequences, its gradient
// and its single steps.
//
//     h_t = f_t h_{t-1} + (1 - f_t) v_t,  f = 1 / (1 + e^-g)
//
// with both f and z = 1 - f to a few ulp of themselves (and of the exponent,
// 2 |g| ulp).  Neither can stand for the other: z = 1 - f has lost its digits
// where f is near 1, and f rounded there would be off by a fixed 2^-25 in every
// step, which a memory of 1 / z steps multiplies; f = 1 - z has lost them where
// f is small, and what should have vanished of a large state stays.
//
// Over a run of tokens the state goes from h to P h + B, where P = prod f and B
// is the run's answer from a zero state; D = 1 - P is its answer to v = 1, so
// accurate where it is small.  Runs are handed on as B and the smaller of P and
// D, and folded as P h + B or h - D h + B: decays stay accurate relative to
// themselves, and the rounding of P near 1 stays within 16 tokens.
// An infinite state stays what it is: the folds of a step in which one occurs are
// made again, since h - D h is no number then.
//
// Bound by memory: every token is read once.  A CTA has 128 bytes of channels
// (4 per lane: 2 bf16 channels, worked on as a pair, or 1 f32) of one chunk of
// 128 tokens, a warp 16 consecutive tokens of it: one walk over them forms the
// gates, and P and B up to every token, which stay in registers; the warps'
// meet in shared memory, a CTA's totals go to the other CTAs of its cluster (as
// many consecutive chunks of the same channels) by asynchronous stores that
// arrive on an mbarrier, every CTA folds them onto the running state, and a
// second walk writes the outputs.  Then the cluster moves on by its chunks.  Tiles
// arrive by TMA, steps ahead; two CTAs per SM fill each other's waits.  Tensors
// that TMA cannot describe arrive row by row, by copies of the 16-byte pieces
// that hold a row, and a lane reads its channels at the row's offset in them.
// Folds go in the order of the tokens: results do not depend on timing.  Chunks
// wholly past a sequence's end are neither read nor walked, only blanked.
//
// The gradient walks the chunks from the end with c_t = f_t lam_t, the
// gradient that leaves token t for h_{t-1}: lam_t = dy_t + c_{t+1}, so a run
// takes c to P c + E with the same P; h_{t-1} is walked forward again from the
// chunk's stored state.
//
// Sequences of up to 16 tokens (a decoder's step) need none of this: a warp
// walks its lanes' channels from global memory.
//
// Measured (bf16; bytes that have to move at the measured copy rate take 62,
// 103, 123 and 205 us): 4 x 8192 x 2048 tokens x channels 78 us, its gradient
// 141; 1 x 131072 x 1024 190 and 350, where the cluster's exchange in every step
// shows; rows that TMA cannot describe (4 x 8192 x 2047) 132 and 240, bound by
// the shared-memory reads at odd offsets and the halved stores (f32 there 165 and
// 335); one token of 64
// sequences x 4096 channels 2.2.  What is left in the first two is the gates'
// exponential and reciprocal and the walks' dependent steps, two CTAs' worth
// of them per SM.
#include <cstring>
#include <type_traits>

#include "block_common.cuh"
#include "common.cuh"
#include "tc_shared.cuh"

namespace hx {
namespace {

using namespace umma;

constexpr int kChunk = HELIX_GATED_CHUNK;
constexpr int kTok = 16;                  // tokens of a warp
constexpr int kWarps = kChunk / kTok;
constexpr int kThreads = 32 * kWarps;
constexpr int kMaxCluster = 8;
constexpr int kAhead = 4;                 // tokens of v that the gradient reads at once (an even number)
// Warps that form a CTA's total and hand it to its cluster (1 x 131072 x 1024
// bf16, gradient: 348 us with two, 352 with four, 379 with eight).
constexpr int kSenders = 2;
constexpr int kTileBytes = kChunk * 128;  // 128 tokens x 128 bytes of channels
constexpr int kFewWarps = 8;              // of a CTA of the few-token kernels

// How a kernel reaches the token tensors.
enum Access { kTma, kWord, kHalf };       // tiles; rows at multiples of 4 bytes, or of 2

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
    static __device__ __forceinline__ V mul(V a, V b) { return f2_mul(a, b); }
    static __device__ __forceinline__ V unpack(uint32_t w) { return f2_of_bf16x2(w); }
    static __device__ __forceinline__ uint32_t pack(V v) {
        float a[2];
        to(v, a);
        return bf16x2(a[0], a[1]);
    }
    static constexpr uint32_t kInf = 0x7f807f80u;
};

// f = sigmoid(g) and z = 1 - f, each to (12 + 2 |g|) 2^-24 of itself (the
// exponent's rounding, the exponential, the reciprocal): with t = e^g, z = 1 /
// (1 + t) and f = t z.  f is zero below 2^-126.  t stops at 2^126, where the
// reciprocal is still normal: larger g have z = 2^-126 and f = 1 exactly, so
// that +infinity with v = 0, which tokens past the end are given, leaves every
// state as it is.
template <typename T>
__device__ __forceinline__ void gate(typename Lane<T>::V g, typename Lane<T>::V& f, typename Lane<T>::V& z) {
    using L = Lane<T>;
    float t[L::kN], r[L::kN];
    L::to(L::mul(g, L::splat(1.4426950408889634f)), t);
#pragma unroll
    for (int e = 0; e < L::kN; ++e)
        asm("ex2.approx.ftz.f32 %0, %0;\n\tmin.NaN.f32 %0, %0, 0f7e800000;" : "+f"(t[e]));
    const typename L::V tv = L::of(t);
    L::to(L::add(tv, L::splat(1.0f)), r);
#pragma unroll
    for (int e = 0; e < L::kN; ++e) asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(r[e]));
    z = L::of(r);
    f = L::mul(tv, z);
}
// The smaller one, m = t / (1 + t) with t = e^-|g|, down to 2^-134 on both
// sides: the exponential gives 2^8 t, whose normal values reach that far, and the
// product with 2^-8 keeps subnormal ones.
template <typename T>
__device__ __forceinline__ typename Lane<T>::V gate_min(const float (&g)[Lane<T>::kN]) {
    using L = Lane<T>;
    float t[L::kN], r[L::kN];
#pragma unroll
    for (int e = 0; e < L::kN; ++e) {
        t[e] = fmaf(-fabsf(g[e]), 1.4426950408889634f, 8.0f);
        asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(t[e]));
    }
    const typename L::V tv = L::mul(L::of(t), L::splat(0x1p-8f));
    L::to(L::add(tv, L::splat(1.0f)), r);
#pragma unroll
    for (int e = 0; e < L::kN; ++e) asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(r[e]));
    return L::mul(tv, L::of(r));
}
// Both from it, for the gradient, whose dg has f z as a factor.
template <typename T>
__device__ __forceinline__ void gate_both(typename Lane<T>::V g, typename Lane<T>::V& f, typename Lane<T>::V& z) {
    using L = Lane<T>;
    float x[L::kN], m[L::kN], o[L::kN], a[L::kN], b[L::kN];
    L::to(g, x);
    const typename L::V mv = gate_min<T>(x);
    L::to(mv, m), L::to(L::fma(mv, L::splat(-1.0f), L::splat(1.0f)), o);
#pragma unroll
    for (int e = 0; e < L::kN; ++e) {
        a[e] = x[e] >= 0.0f ? o[e] : m[e];
        b[e] = x[e] >= 0.0f ? m[e] : o[e];
    }
    f = L::of(a), z = L::of(b);
}
// What is left of a state after a step, or a run of them, as one number: the
// smaller of the decay P = prod f and D = 1 - P, which fixes both with full
// precision: P itself, or -D.  In the sign, not in a comparison with zero: what
// keeps all of a state is -0.
__device__ __forceinline__ bool keeps(float c) { return __float_as_int(c) < 0; }

// Of a step.
template <typename T>
__device__ __forceinline__ typename Lane<T>::V gate_decay(typename Lane<T>::V g) {
    using L = Lane<T>;
    float x[L::kN], c[L::kN];
    L::to(g, x);
    L::to(gate_min<T>(x), c);
#pragma unroll
    for (int e = 0; e < L::kN; ++e) c[e] = copysignf(c[e], -x[e]);
    return L::of(c);
}
// f x and z x; f h + z v; z f.  Where f is near 1 it is not rounded: over the
// 1 / z steps of its memory that would add up.  (x - z x and h - v are no numbers
// where x, h or v is infinite, and h - v need not be one where it is only large:
// then the products that the formula has.)
constexpr float kInfinity = __builtin_huge_valf();
__device__ __forceinline__ bool finite(float x) { return fabsf(x) < kInfinity; }
__device__ __forceinline__ float f_of(float c) { return keeps(c) ? 1.0f + c : c; }
__device__ __forceinline__ float z_of(float c) { return keeps(c) ? -c : 1.0f - c; }
__device__ __forceinline__ float kept(float c, float x) {
    return finite(x) ? fmaf(c, x, keeps(c) ? x : 0.0f) : f_of(c) * x;
}
__device__ __forceinline__ float taken(float c, float x) {
    return finite(x) ? (keeps(c) ? -c * x : fmaf(-c, x, x)) : z_of(c) * x;
}
__device__ __forceinline__ float moved(float c, float h, float v) { return fmaf(c, h - v, keeps(c) ? h : v); }
__device__ __forceinline__ float moved_any(float c, float h, float v) {
    return finite(h - v) ? moved(c, h, v) : fmaf(f_of(c), h, z_of(c) * v);
}
__device__ __forceinline__ float slope(float c) { return fmaf(-c, c, fabsf(c)); }

// Of a run with P and D.  (Packed arithmetic has no negation and no absolute
// value; single selects have both for nothing.)
template <typename L>
__device__ __forceinline__ typename L::V decay_of(typename L::V p, typename L::V d) {
    float a[L::kN], b[L::kN];
    L::to(p, a), L::to(d, b);
#pragma unroll
    for (int e = 0; e < L::kN; ++e) a[e] = a[e] > 0.5f ? -fabsf(b[e]) : a[e];
    return L::of(a);
}
// P h + b.
template <typename L>
__device__ __forceinline__ typename L::V fold(typename L::V h, typename L::V c, typename L::V b) {
    float x[L::kN], d[L::kN];
    L::to(h, x), L::to(c, d);
#pragma unroll
    for (int e = 0; e < L::kN; ++e) x[e] = keeps(d[e]) ? x[e] : 0.0f;
    return L::add(L::fma(c, h, L::of(x)), b);
}
// The same for infinite h too, which stay what they are (P > 0, even where it
// is zero in fp32).
template <typename L>
__device__ __forceinline__ typename L::V fold_any(typename L::V h, typename L::V c, typename L::V b) {
    float x[L::kN], d[L::kN], y[L::kN];
    L::to(h, x), L::to(c, d), L::to(b, y);
#pragma unroll
    for (int e = 0; e < L::kN; ++e)
        x[e] = fabsf(x[e]) == kInfinity ? x[e] + y[e] : fmaf(d[e], x[e], keeps(d[e]) ? x[e] : 0.0f) + y[e];
    return L::of(x);
}
// P of a state h, 1 where that is infinite.
template <typename L>
__device__ __forceinline__ typename L::V unless_infinite(typename L::V p, typename L::V h) {
    float a[L::kN], x[L::kN];
    L::to(p, a), L::to(h, x);
#pragma unroll
    for (int e = 0; e < L::kN; ++e) a[e] = fabsf(x[e]) == kInfinity ? 1.0f : a[e];
    return L::of(a);
}
// Whether one of the lane's n channels is infinite or NaN.  No fold makes
// either finite again, so it is enough to look at the last of a row of them.
template <typename L>
__device__ __forceinline__ bool lost(typename L::V h, int n) {
    float x[L::kN];
    L::to(h, x);
    bool any = false;
#pragma unroll
    for (int e = 0; e < L::kN; ++e) any = any || (e < n && !finite(x[e]));
    return any;
}
// P and -D of several runs, one after the other (D counts only where every
// run keeps more than half, and there each has -D).
template <typename L>
struct Runs {
    typename L::V p = L::splat(1.0f), nd = L::splat(0.0f), b = nd;
    // kAny: with infinite b's too.
    template <bool kAny>
    __device__ __forceinline__ void add(typename L::V c, typename L::V bc) {
        float k[L::kN], d[L::kN];
        L::to(L::add(c, L::splat(1.0f)), k), L::to(c, d);
#pragma unroll
        for (int e = 0; e < L::kN; ++e) k[e] = keeps(d[e]) ? k[e] : d[e];
        p = L::mul(p, L::of(k));
        nd = L::add(L::fma(nd, c, nd), c);
        b = kAny ? fold_any<L>(b, c, bc) : fold<L>(b, c, bc);
    }
    __device__ __forceinline__ typename L::V decay() const { return decay_of<L>(p, nd); }
};

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
__device__ __forceinline__ void ld_state(const float* p, int n, float (&a)[L::kN]) {
#pragma unroll
    for (int e = 0; e < L::kN; ++e) a[e] = p && e < n ? __ldg(p + e) : 0.0f;
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

__device__ __forceinline__ uint32_t align128(const uint8_t* p) { return (smem_u32(p) + 127u) & ~127u; }
__device__ __forceinline__ uint32_t lds_half(uint32_t a) {
    unsigned short v;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(a));
    return v;
}
// Shared memory by its 32-bit address: 64-bit generic addresses cost two more
// instructions an access.
__device__ __forceinline__ uint32_t lds(uint32_t a) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a));
    return v;
}

__device__ __forceinline__ void sts(uint32_t a, float v) {
    asm volatile("st.shared.f32 [%0], %1;" ::"r"(a), "f"(v) : "memory");
}

// How a CTA cuts its tile: rows of LW lanes' channels (32, or 16 to make twice
// as many CTAs of few channels), a run of 16 tokens for each LW lanes.
template <int LW>
struct Cut {
    static constexpr int kRuns = 32 / LW;                    // runs of a warp
    static constexpr int kTokens = kWarps * kRuns * kTok;    // of a CTA and step
    static constexpr int kRow = 4 * LW;                      // bytes
    static_assert(kTokens * kRow == kTileBytes, "tile");
    // Copied rows: at an offset of up to 15 in a slot; the runs of a warp half
    // the banks apart.
    static constexpr int kSlot = kRow + 16;
    static constexpr int kRun = kTok * kSlot + (LW == 16 ? 64 : 0);
    static constexpr int kRowTile = kWarps * kRuns * kRun;
    // Word i of tensor k, from the lane's first word.
    static __host__ __device__ constexpr uint32_t word(int k, int i) { return (uint32_t)(k * kTileBytes + i * kRow); }
};

// Where a thread is: its group of channels, and its run of a step's tokens.
template <typename T, int LW>
struct Place {
    int warp, lane, l, run, rank, seq, c0, n, len;
    __device__ __forceinline__ Place(const GatedParams& p) {
        constexpr int N = Lane<T>::kN, CB = LW * N;
        warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0);
        lane = threadIdx.x & 31;
        l = lane % LW;
        run = warp * Cut<LW>::kRuns + lane / LW;
        rank = (int)(blockIdx.x % (unsigned)p.cluster);
        const int slabs = (p.n_chan + CB - 1) / CB;
        const unsigned group = blockIdx.x / (unsigned)p.cluster;
        seq = (int)(group / (unsigned)slabs);
        c0 = (int)(group % (unsigned)slabs) * CB + N * l;
        n = max(0, min(N, p.n_chan - c0));
        len = length_of(p, seq);
    }
    __device__ __forceinline__ int slab0() const { return c0 - Lane<T>::kN * l; }
    // Whether every token and channel of the warp counts, in the step at `base`.
    __device__ __forceinline__ bool whole(const GatedParams& p, int base) const {
        return base + (warp + 1) * Cut<LW>::kRuns * kTok <= len && slab0() + LW * Lane<T>::kN <= p.n_chan;
    }
};

// Zeros for the lane's channels of a run's tokens from t0 on.
template <typename T, Access A>
__device__ __forceinline__ void blank(T* row, int64_t s_tok, int t0, int n_tok, int n) {
#pragma unroll
    for (int i = 0; i < kTok; ++i)
        if (n > 0 && t0 + i < n_tok) st_raw<T, A>(row + (t0 + i) * s_tok, n, 0u);
}

// The values of the warp's first and last run, where it has two.
__device__ __forceinline__ float of_lane(float v, int lane) { return __shfl_sync(0xffffffffu, v, lane); }
__device__ __forceinline__ uint64_t of_lane(uint64_t v, int lane) {
    return __shfl_sync(0xffffffffu, (unsigned long long)v, lane);
}

// The warps' (D, B) of a step, and the totals of the cluster's CTAs with the
// mbarrier they arrive on; two steps' worth, since a warp may be a step ahead
// of another (the gradient's warps are not, and the 6 KB decide whether two of
// its CTAs fit an SM).
template <typename V, int K, int kSteps = 2>
struct Meet {
    V        warp[kSteps][K][kWarps][32];
    V        total[2][2][kMaxCluster][32];
    uint64_t arrived[2];
    uint32_t lost;  // a warp's answer has been infinite or NaN in this or an earlier step
};

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t in_rank(const void* p, int rank) {
    uint32_t a;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
    return a;
}
// Store to another CTA's shared memory; its mbarrier counts the bytes.
__device__ __forceinline__ void st_async(uint32_t at, uint64_t v, uint32_t bar) {
    asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.b64 [%0], %1, [%2];" ::"r"(at), "l"(v),
                 "r"(bar)
                 : "memory");
}
__device__ __forceinline__ void st_async(uint32_t at, float v, uint32_t bar) {
    asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.b32 [%0], %1, [%2];" ::"r"(at),
                 "r"(__float_as_uint(v)), "r"(bar)
                 : "memory");
}
// Asynchronous copy of 16 bytes to shared memory.
__device__ __forceinline__ void copy16(uint32_t to, uintptr_t from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ bool try_wait_cluster(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}

template <int N>
struct Size {
    __device__ __forceinline__ constexpr operator int() const { return N; }
};
// The body with the cluster's size as a constant, so that its loop's shared
// loads are all issued before the first is looked at.
template <typename F>
__device__ __forceinline__ void by_cluster(int size, F body) {
    static_assert(kMaxCluster == 8, "");
    if (size == 8)
        body(Size<8>{});
    else if (size == 4)
        body(Size<4>{});
    else
        body(Size<2>{});
}

struct GatedMaps {
    CUtensorMap in[3];  // g, v, dy
};

// What the threads of a CTA share in the walk over its chunks: the tiles of
// the K input tensors, kStages steps of them, and the meetings of a step.
template <typename T, Access A, int K, int kStages, int LW, typename M>
struct Walk {
    using L = Lane<T>;
    using V = typename L::V;
    const GatedMaps&   maps;
    const GatedParams& p;
    const Place<T, LW>& at;
    uint32_t           base;  // shared-memory address of the tiles
    uint64_t*          full;
    M*                 meet;
    int                steps;  // that hold tokens before the sequence's end
    bool               alive = true;

    // Copied rows: tensor k's of the sequence, at the slab's first channel, and their pitch.
    const T* rows[A == kTma ? 1 : K];
    int64_t  pitch[A == kTma ? 1 : K];

    // Tiles.  The lane's words of step s.
    __device__ __forceinline__ uint32_t mine(int s) const {
        constexpr int kTile = A == kTma ? kTileBytes : Cut<LW>::kRowTile;
        constexpr int kRun = A == kTma ? kTok * Cut<LW>::kRow : Cut<LW>::kRun;
        return base + (uint32_t)((s % kStages) * K * kTile + at.run * kRun + at.l * 4);
    }
    // Offset in its 16-byte piece of the run's first row of a step's tensor,
    // and what a row adds to it.
    struct Shift {
        uint32_t first, step;
    };
    __device__ __forceinline__ Shift shift(int k, int t0) const {
        if (A == kTma) return {0u, 0u};
        return {(uint32_t)(reinterpret_cast<uintptr_t>(rows[k] + t0 * pitch[k])) & 15u,
                (uint32_t)(pitch[k] * (int64_t)sizeof(T)) & 15u};
    }
    // The lane's channels of token i of tensor k.
    __device__ __forceinline__ uint32_t word_at(uint32_t my, const Shift& sh, int k, int i) const {
        if (A == kTma) return my + Cut<LW>::word(k, i);
        const uint32_t off = (sh.first + i * sh.step) & 15u;
        return my + (uint32_t)(k * Cut<LW>::kRowTile + i * Cut<LW>::kSlot) + off;
    }
    __device__ __forceinline__ uint32_t get(uint32_t my, const Shift& sh, int k, int i) const {
        const uint32_t a = word_at(my, sh, k, i);
        return A != kHalf ? lds(a) : lds_half(a) | lds_half(a + 2) << 16;
    }
    // The lane's tokens past the sequence's end become ones that leave every
    // state as it is: g = +infinity, v = dy = 0.  (In the tiles, so that the
    // walks have one form, whose registers need no merging.)
    __device__ __forceinline__ void close(uint32_t my, int t0, const Shift& sg, const Shift& sv, const Shift& sdy) const {
#pragma unroll 1
        for (int i = max(0, at.len - t0); i < kTok; ++i) {
            put(my, sg, 0, i, L::kInf);
            put(my, sv, 1, i, 0u);
            if (K > 2) put(my, sdy, 2, i, 0u);
        }
        if (A == kTma) fence_async_smem();
    }
    __device__ __forceinline__ void put(uint32_t my, const Shift& sh, int k, int i, uint32_t w) const {
        const uint32_t a = word_at(my, sh, k, i);
        if (A != kHalf) {
            asm volatile("st.shared.u32 [%0], %1;" ::"r"(a), "r"(w) : "memory");
        } else {
            asm volatile("st.shared.u16 [%0], %1;" ::"r"(a), "h"((unsigned short)w) : "memory");
            asm volatile("st.shared.u16 [%0], %1;" ::"r"(a + 2), "h"((unsigned short)(w >> 16)) : "memory");
        }
    }
    // The gates of the lane's token i of step s, put aside where registers are
    // short: into the words of the first two tensors' tiles that the lane has
    // read, or beside copied rows, whose words may be at odd addresses.  Runs
    // of narrow tiles lie on the same banks, so one of a warp's two takes tokens
    // i ^ 1 (1 x 131072 x 1024 bf16: 366 -> 352 us).
    __device__ __forceinline__ uint32_t gate_at(int s, int i) const {
        if (A == kTma) {
            const int turn = LW == 16 ? at.run & 1 : 0;
            return mine(s) + Cut<LW>::word(0, i) + (i & 1 ? -turn : turn) * Cut<LW>::kRow;
        }
        return base + (uint32_t)(kStages * K * Cut<LW>::kRowTile +
                                 ((at.run * kTok + i) * LW + at.l) * (int)sizeof(float) * L::kN);
    }
    __device__ __forceinline__ void put_gate(int s, int i, V f) const {
        const uint32_t to = gate_at(s, i);
        float a[L::kN];
        L::to(f, a);
        if constexpr (L::kN == 1) {
            sts(to, a[0]);
        } else if constexpr (A == kTma) {
            sts(to, a[0]);
            sts(to + kTileBytes, a[1]);
        } else {
            asm volatile("st.shared.v2.f32 [%0], {%1, %2};" ::"r"(to), "f"(a[0]), "f"(a[1]) : "memory");
        }
    }
    __device__ __forceinline__ V take_gate(int s, int i) const {
        const uint32_t from = gate_at(s, i);
        float a[L::kN];
        if constexpr (L::kN == 1) {
            a[0] = __uint_as_float(lds(from));
        } else if constexpr (A == kTma) {
            a[0] = __uint_as_float(lds(from));
            a[1] = __uint_as_float(lds(from + kTileBytes));
        } else {
            asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(a[0]), "=f"(a[1]) : "r"(from));
        }
        return L::of(a);
    }
    __device__ __forceinline__ bool issuer() const { return A == kTma && threadIdx.x == kThreads - 1; }
    // One thread: step s's tiles (chunk `chunk`) start to arrive.
    __device__ __forceinline__ void load(int s, int chunk) const {
        uint64_t* bar = &full[s % kStages];
        mbar_expect_tx(bar, K * kTileBytes);
#pragma unroll
        for (int k = 0; k < K; ++k)
            tma_load_3d(base + (uint32_t)(((s % kStages) * K + k) * kTileBytes), &maps.in[k], bar, at.slab0(),
                        chunk * Cut<LW>::kTokens, at.seq);
    }
    // Every warp: step s's rows of its runs (none past the last step) start to
    // arrive, one group of copies: the 16-byte pieces that hold a row's
    // channels, each of which holds one that exists.  A row's whole pieces go
    // to as many lanes, the one that an offset adds to one lane per row.
    __device__ __forceinline__ void copy_rows(int s, int chunk) const {
        if constexpr (A != kTma) {
            constexpr int kPieces = Cut<LW>::kRow / 16, kAtOnce = 32 / kPieces, kRows = Cut<LW>::kRuns * kTok;
            if (s < steps) {
                const int t0 = chunk * Cut<LW>::kTokens + at.warp * kRows;
                const uint32_t to = mine(s) - (uint32_t)((at.run % Cut<LW>::kRuns) * Cut<LW>::kRun + at.l * 4);
                const int width = min(LW * Lane<T>::kN, p.n_chan - at.slab0()) * (int)sizeof(T);
                auto piece = [&](int k, const T* row, int r, int b) {  // the one at byte b of row r
                    const uintptr_t a = reinterpret_cast<uintptr_t>(row);
                    if (t0 + r < at.len && b < (int)(a & 15) + width)
                        copy16(to + (uint32_t)(k * Cut<LW>::kRowTile + r / kTok * Cut<LW>::kRun +
                                               r % kTok * Cut<LW>::kSlot + b),
                               (a & ~uintptr_t(15)) + b);
                };
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    const T* row = rows[k] + (t0 + at.lane / kPieces) * pitch[k];
#pragma unroll
                    for (int r = 0; r < kRows; r += kAtOnce, row += kAtOnce * pitch[k])
                        piece(k, row, r + at.lane / kPieces, at.lane % kPieces * 16);
                    if (at.lane < kRows) piece(k, rows[k] + (t0 + at.lane) * pitch[k], at.lane, Cut<LW>::kRow);
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        }
    }
    // Before the warps meet: whether the lane's is infinite or NaN; and after,
    // whether one was.
    __device__ __forceinline__ void note(V t) const {
        if (lost<L>(t, at.n)) *const_cast<volatile uint32_t*>(&meet->lost) = 1;
    }
    __device__ __forceinline__ bool noted() const { return *const_cast<const volatile uint32_t*>(&meet->lost) != 0; }
    __device__ __forceinline__ void gave_up() {
        alive = false;
        if (p.fault) atomicCAS(p.fault, 0u, (unsigned)kFaultGated);
    }
    __device__ __forceinline__ void wait_tiles(int s) {
        if (A == kTma) {
            if (alive && !mbar_wait(&full[s % kStages], (uint32_t)((s / kStages) & 1), tc::kWaitBudget)) gave_up();
        } else {
            asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
        }
        __syncwarp();
    }
    __device__ __forceinline__ void begin() {
        if (threadIdx.x == kThreads - 1) {
#pragma unroll
            for (int k = 0; k < kStages; ++k) mbar_init(&full[k], 1);
            mbar_init(&meet->arrived[0], 1);
            mbar_init(&meet->arrived[1], 1);
            meet->lost = 0;
            fence_mbar_init();
        }
        __syncthreads();
        if (p.cluster > 1) cluster_sync();  // no CTA writes to another before that one's barriers stand
    }
    // The totals of step s to every CTA of the cluster, of the warps' decays c
    // and answers t, taken from warp `from` on in steps of `turn`.  Formed and
    // sent by the first warps of that order (nth: this one's place), which have
    // the least to fold once the others' totals are there.
    __device__ __forceinline__ void send(int s, int nth, const V (&c)[kWarps][32], const V (&t)[kWarps][32], int from,
                                         int turn) {
        const int b = s & 1, senders = min(p.cluster, kSenders);
        if (at.warp == 0 && at.lane == 0)
            mbar_expect_tx(&meet->arrived[b], (uint32_t)(p.cluster * 2 * 32 * sizeof(V)));
        if (nth < senders) {
            Runs<L> all;
            if (noted()) {
#pragma unroll 1
                for (int w = 0; w < kWarps; ++w)
                    all.template add<true>(c[from + turn * w][at.lane], t[from + turn * w][at.lane]);
            } else {
#pragma unroll
                for (int w = 0; w < kWarps; ++w)
                    all.template add<false>(c[from + turn * w][at.lane], t[from + turn * w][at.lane]);
            }
            const V d = all.decay();
            for (int r = nth; r < p.cluster; r += senders) {
                const uint32_t bar = in_rank(&meet->arrived[b], r);
                st_async(in_rank(&meet->total[b][0][at.rank][at.lane], r), d, bar);
                st_async(in_rank(&meet->total[b][1][at.rank][at.lane], r), all.b, bar);
            }
        }
    }
    __device__ __forceinline__ void receive(int s) {
        if (alive) {
            uint64_t*      bar = &meet->arrived[s & 1];
            const uint32_t parity = (uint32_t)((s >> 1) & 1);
            if (!try_wait_cluster(bar, parity)) {
                const long long t0 = clock64();
                while (!try_wait_cluster(bar, parity))
                    if (clock64() - t0 > tc::kWaitBudget) {
                        gave_up();
                        break;
                    }
            }
        }
        __syncwarp();
    }
    __device__ __forceinline__ void end() {
        // whatever became of the other waits, the loads land
        if (issuer())
            for (int s = max(0, steps - kStages); s < steps; ++s)
                mbar_wait(&full[s % kStages], (uint32_t)((s / kStages) & 1), tc::kWaitBudget);
        if (A != kTma) asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncwarp();
        if (p.cluster > 1) cluster_sync();  // no CTA leaves while another may store to it
    }
};

template <typename T, Access A, int kStages, int LW>
__global__ void __launch_bounds__(kThreads, 2)
    gated_kernel(const __grid_constant__ GatedMaps maps, const __grid_constant__ GatedParams p) {
    using L = Lane<T>;
    using V = typename L::V;
    extern __shared__ uint8_t smem_raw[];
    using M = Meet<V, 2>;
    __shared__ M meet;
    __shared__ uint64_t full[kStages];

    const Place<T, LW> at(p);
    const int R = p.cluster, warp = at.warp, lane = at.lane, n = at.n;
    const int steps = ((at.len + Cut<LW>::kTokens - 1) / Cut<LW>::kTokens + R - 1) / R;
    Walk<T, A, 2, kStages, LW, M> walk{maps, p, at, align128(smem_raw), full, &meet, steps};
    auto chunk_of = [&](int s) { return s * R + at.rank; };
    walk.begin();
    if constexpr (A != kTma) {
        walk.rows[0] = static_cast<const T*>(p.g) + (int64_t)at.seq * p.seq_g + at.slab0(), walk.pitch[0] = p.s_g;
        walk.rows[1] = static_cast<const T*>(p.v) + (int64_t)at.seq * p.seq_v + at.slab0(), walk.pitch[1] = p.s_v;
    }
    for (int s = 0; s < kStages; ++s) {
        if (walk.issuer() && s < steps) walk.load(s, chunk_of(s));
        walk.copy_rows(s, chunk_of(s));
    }
    __syncwarp();

    V h = ld_state<L>(p.h0 ? p.h0 + (int64_t)at.seq * p.seq_h0 + at.c0 : nullptr, n);
    for (int s = 0; s < steps; ++s) {
        const int base = chunk_of(s) * Cut<LW>::kTokens, t0 = base + at.run * kTok, b = s & 1;
        const uint32_t my = walk.mine(s);
        const bool whole = at.whole(p, base);
        // P and B of the run up to each token: h_t = P h + B
        V ph[kTok], hb[kTok], P = L::splat(1.0f), D = L::splat(0.0f), B = D;
        const auto shift_g = walk.shift(0, t0), shift_v = walk.shift(1, t0);
        walk.wait_tiles(s);
        if (!whole) walk.close(my, t0, shift_g, shift_v, shift_g);
#pragma unroll
        for (int i = 0; i < kTok; ++i) {
            V f, z;
            gate<T>(L::unpack(walk.get(my, shift_g, 0, i)), f, z);
            ph[i] = P = L::mul(P, f);
            D = L::fma(f, D, z);
            hb[i] = B = L::fma(f, B, L::mul(z, L::unpack(walk.get(my, shift_v, 1, i))));
        }
        if (A != kTma) {  // the warp is done with its rows
            __syncwarp();
            walk.copy_rows(s + kStages, chunk_of(s + kStages));
        }
        V c0 = decay_of<L>(P, D), b0 = B;  // the warp's first run
        if (LW == 16) {
            const V p0 = of_lane(P, at.l), p1 = of_lane(P, at.l + 16), d0 = of_lane(D, at.l),
                    d1 = of_lane(D, at.l + 16), b1 = of_lane(B, at.l + 16);
            c0 = decay_of<L>(p0, d0), b0 = of_lane(B, at.l);
            P = L::mul(p0, p1);
            D = L::fma(p0, d1, d0);
            B = fold_any<L>(b0, decay_of<L>(p1, d1), b1);
        }
        meet.warp[b][0][warp][lane] = LW == 16 ? decay_of<L>(P, D) : c0;
        meet.warp[b][1][warp][lane] = B;
        walk.note(B);
        __syncthreads();  // and every warp is done with the tiles
        if (walk.issuer() && s + kStages < steps) walk.load(s + kStages, chunk_of(s + kStages));
        __syncwarp();
        const V entry = h;
        V hw = h;
        if (R > 1) {
            walk.send(s, warp, meet.warp[b][0], meet.warp[b][1], 0, 1);
            walk.receive(s);
            by_cluster(R, [&](auto size) {
#pragma unroll
                for (int k = 0; k < size; ++k) {
                    if (k == at.rank) hw = h;
                    h = fold<L>(h, meet.total[b][0][k][lane], meet.total[b][1][k][lane]);
                }
            });
#pragma unroll
            for (int w = 0; w < kWarps - 1; ++w)
                if (w < warp) hw = fold<L>(hw, meet.warp[b][0][w][lane], meet.warp[b][1][w][lane]);
        } else {
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                if (w == warp) hw = h;
                h = fold<L>(h, meet.warp[b][0][w][lane], meet.warp[b][1][w][lane]);
            }
        }
        if (LW == 16 && lane >= 16) hw = fold<L>(hw, c0, b0);
        auto second = [&](auto all, auto infinite) {
            if (p.states && t0 % kChunk == 0 && t0 < p.n_tok)
                st_state<L>(p.states + ((int64_t)at.seq * p.n_chunk + t0 / kChunk) * p.n_chan + at.c0, n, hw);
            T* y = static_cast<T*>(p.y) + (int64_t)at.seq * p.seq_y + at.c0 + (int64_t)t0 * p.s_y;
#pragma unroll
            for (int i = 0; i < kTok; ++i) {
                const bool past = !decltype(all)::value && t0 + i >= at.len;
                const V pi = decltype(infinite)::value ? unless_infinite<L>(ph[i], hw) : ph[i];
                if (decltype(all)::value || (n > 0 && t0 + i < p.n_tok))
                    st_raw<T, A>(y, decltype(all)::value ? L::kN : n, past ? 0u : L::pack(L::fma(pi, hw, hb[i])));
                y += p.s_y;
            }
        };
        if (whole)
            second(std::true_type{}, std::false_type{});
        else
            second(std::false_type{}, std::false_type{});
        // An infinity or a NaN: once more, with folds that keep infinities.  Here,
        // where nothing waits for the answer (before the outputs: 1 x 131072 x 1024
        // bf16 202 us, here 190).
        if (__any_sync(0xffffffffu, lost<L>(h, n))) {
            h = hw = entry;
            if (R > 1) {
#pragma unroll 1
                for (int k = 0; k < R; ++k) {
                    if (k == at.rank) hw = h;
                    h = fold_any<L>(h, meet.total[b][0][k][lane], meet.total[b][1][k][lane]);
                }
            }
            V x = hw;
#pragma unroll 1
            for (int w = 0; w < kWarps; ++w) {
                if (w == warp) hw = x;
                x = fold_any<L>(x, meet.warp[b][0][w][lane], meet.warp[b][1][w][lane]);
            }
            if (R == 1) h = x;
            if (LW == 16 && lane >= 16) hw = fold_any<L>(hw, c0, b0);
            second(std::false_type{}, std::true_type{});
        }
    }
    walk.end();
    for (int k = chunk_of(steps); k * Cut<LW>::kTokens < p.n_tok; k += R) {  // past the sequence's end
        const int t0 = k * Cut<LW>::kTokens + at.run * kTok;
        blank<T, A>(static_cast<T*>(p.y) + (int64_t)at.seq * p.seq_y + at.c0, p.s_y, t0, p.n_tok, n);
        if (p.states && t0 % kChunk == 0 && t0 < p.n_tok)
            st_state<L>(p.states + ((int64_t)at.seq * p.n_chunk + t0 / kChunk) * p.n_chan + at.c0, n, h);
    }
    // Every CTA holds the last state.  In place of h0 is safe: each has read
    // h0 before the cluster's last barrier.
    if (at.rank == 0 && warp == 0 && lane < LW) st_state<L>(p.h1 + (int64_t)at.seq * p.seq_h1 + at.c0, n, h);
}

template <typename T, Access A, int kStages, int LW>
__global__ void __launch_bounds__(kThreads, 2)
    gated_grad_kernel(const __grid_constant__ GatedMaps maps, const __grid_constant__ GatedParams p) {
    using L = Lane<T>;
    using V = typename L::V;
    extern __shared__ uint8_t smem_raw[];
    using M = Meet<V, 3, 1>;
    __shared__ M meet;
    __shared__ uint64_t full[kStages];

    const Place<T, LW> at(p);
    const int R = p.cluster, warp = at.warp, lane = at.lane, n = at.n;
    const int steps = ((at.len + Cut<LW>::kTokens - 1) / Cut<LW>::kTokens + R - 1) / R;
    Walk<T, A, 3, kStages, LW, M> walk{maps, p, at, align128(smem_raw), full, &meet, steps};
    auto chunk_of = [&](int s) { return (steps - 1 - s) * R + at.rank; };  // from the end
    walk.begin();
    if constexpr (A != kTma) {
        walk.rows[0] = static_cast<const T*>(p.g) + (int64_t)at.seq * p.seq_g + at.slab0(), walk.pitch[0] = p.s_g;
        walk.rows[1] = static_cast<const T*>(p.v) + (int64_t)at.seq * p.seq_v + at.slab0(), walk.pitch[1] = p.s_v;
        walk.rows[2] = static_cast<const T*>(p.dy) + (int64_t)at.seq * p.seq_dy + at.slab0(), walk.pitch[2] = p.s_dy;
    }
    for (int s = 0; s < kStages; ++s) {
        if (walk.issuer() && s < steps) walk.load(s, chunk_of(s));
        walk.copy_rows(s, chunk_of(s));
    }
    __syncwarp();

    V c = ld_state<L>(p.dh1 ? p.dh1 + (int64_t)at.seq * p.seq_dh1 + at.c0 : nullptr, n);
    for (int s = 0; s < steps; ++s) {
        const int base = chunk_of(s) * Cut<LW>::kTokens, t0 = base + at.run * kTok, b = s & 1;
        const uint32_t my = walk.mine(s);
        const bool whole = at.whole(p, base);
        float entry[L::kN];  // the chunk's state; looked at after the warps have met
        const int64_t chunk = (int64_t)at.seq * p.n_chunk + t0 / kChunk;
        ld_state<L>(t0 < p.n_tok ? p.states + chunk * p.n_chan + at.c0 : nullptr, n, entry);
        const auto shift_g = walk.shift(0, t0), shift_v = walk.shift(1, t0), shift_dy = walk.shift(2, t0);
        V z[kTok], q[kTok], P = L::splat(1.0f), D = L::splat(0.0f), B = D, E = D;  // q: f, at first
        walk.wait_tiles(s);
        if (!whole) walk.close(my, t0, shift_g, shift_v, shift_dy);
#pragma unroll
        for (int i = 0; i < kTok; ++i) {
            gate_both<T>(L::unpack(walk.get(my, shift_g, 0, i)), q[i], z[i]);
            P = L::mul(P, q[i]);
            D = L::fma(q[i], D, z[i]);
            B = L::fma(q[i], B, L::mul(z[i], L::unpack(walk.get(my, shift_v, 1, i))));
        }
#pragma unroll
        for (int i = kTok - 1; i >= 0; --i) E = L::mul(q[i], L::add(L::unpack(walk.get(my, shift_dy, 2, i)), E));
        V c0 = decay_of<L>(P, D), b0 = B, c1 = c0, e1 = E;  // the warp's first run, and its last
        if (LW == 16) {
            const V p0 = of_lane(P, at.l), p1 = of_lane(P, at.l + 16), d0 = of_lane(D, at.l),
                    d1 = of_lane(D, at.l + 16), b1 = of_lane(B, at.l + 16), e0 = of_lane(E, at.l);
            c0 = decay_of<L>(p0, d0), c1 = decay_of<L>(p1, d1);
            b0 = of_lane(B, at.l), e1 = of_lane(E, at.l + 16);
            P = L::mul(p0, p1);
            D = L::fma(p0, d1, d0);
            B = fold_any<L>(b0, c1, b1);
            E = fold_any<L>(e1, c0, e0);
        }
        meet.warp[0][0][warp][lane] = LW == 16 ? decay_of<L>(P, D) : c0;
        meet.warp[0][1][warp][lane] = B;
        meet.warp[0][2][warp][lane] = E;
        {  // 0 B + 0 E + 0 entry is NaN where one of them is no finite number
            const V none = L::splat(0.0f);
            walk.note(L::fma(B, none, L::fma(E, none, L::mul(L::of(entry), none))));
        }
        __syncthreads();
        if (R > 1)
            walk.send(s, kWarps - 1 - warp, meet.warp[0][0], meet.warp[0][2], kWarps - 1, -1);
        // h_{t-1} - v_t of the warp's tokens, times the slopes; f into the
        // place of g and v
        V h = L::of(entry);
        auto of_chunk = [&](int w) { return w < warp && w * Cut<LW>::kRuns * kTok >= at.run * kTok / kChunk * kChunk; };
        if (walk.noted()) {
#pragma unroll 1
            for (int w = 0; w < kWarps - 1; ++w)
                if (of_chunk(w)) h = fold_any<L>(h, meet.warp[0][0][w][lane], meet.warp[0][1][w][lane]);
            if (LW == 16 && lane >= 16) h = fold_any<L>(h, c0, b0);
        } else {
#pragma unroll
            for (int w = 0; w < kWarps - 1; ++w)
                if (of_chunk(w)) h = fold<L>(h, meet.warp[0][0][w][lane], meet.warp[0][1][w][lane]);
            if (LW == 16 && lane >= 16) h = fold<L>(h, c0, b0);
        }
#pragma unroll
        for (int i0 = 0; i0 < kTok; i0 += kAhead) {
            uint32_t vw[kAhead];  // read before the first gate is written, which reads do not pass
#pragma unroll
            for (int i = 0; i < kAhead; ++i) vw[i] = walk.get(my, shift_v, 1, i0 + i);
#pragma unroll
            for (int i = i0; i < i0 + kAhead; ++i) {
                const V v = L::unpack(vw[i - i0]), f = q[i], off = L::fma(v, L::splat(-1.0f), h);
                walk.put_gate(s, i, f);
                q[i] = L::mul(L::mul(z[i], f), off);
                h = L::fma(f, h, L::mul(z[i], v));
            }
        }
        const V c_in = c;
        V cw = c;
        if (R > 1) {
            walk.receive(s);
            by_cluster(R, [&](auto size) {
#pragma unroll
                for (int k = size - 1; k >= 0; --k) {
                    if (k == at.rank) cw = c;
                    c = fold<L>(c, meet.total[b][0][k][lane], meet.total[b][1][k][lane]);
                }
            });
#pragma unroll
            for (int w = kWarps - 1; w > 0; --w)
                if (w > warp) cw = fold<L>(cw, meet.warp[0][0][w][lane], meet.warp[0][2][w][lane]);
        } else {
#pragma unroll
            for (int w = kWarps - 1; w >= 0; --w) {
                if (w == warp) cw = c;
                c = fold<L>(c, meet.warp[0][0][w][lane], meet.warp[0][2][w][lane]);
            }
        }
        if (LW == 16 && lane < 16) cw = fold<L>(cw, c1, e1);
        auto second = [&](auto all) {
            T* dg = static_cast<T*>(p.dg) + (int64_t)at.seq * p.seq_dg + at.c0 + (int64_t)(t0 + kTok - 1) * p.s_dg;
            T* dv = static_cast<T*>(p.dv) + (int64_t)at.seq * p.seq_dv + at.c0 + (int64_t)(t0 + kTok - 1) * p.s_dv;
#pragma unroll
            for (int i = kTok - 1; i >= 0; --i) {
                const bool past = !decltype(all)::value && t0 + i >= at.len;
                const V lam = L::add(L::unpack(walk.get(my, shift_dy, 2, i)), cw);
                if (decltype(all)::value || (n > 0 && t0 + i < p.n_tok)) {
                    const int k = decltype(all)::value ? L::kN : n;
                    st_raw<T, A>(dg, k, past ? 0u : L::pack(L::mul(lam, q[i])));
                    st_raw<T, A>(dv, k, past ? 0u : L::pack(L::mul(z[i], lam)));
                }
                dg -= p.s_dg, dv -= p.s_dv;
                cw = L::mul(walk.take_gate(s, i), lam);
            }
        };
        if (whole)
            second(std::true_type{});
        else
            second(std::false_type{});
        // as in the forward walk
        if (__any_sync(0xffffffffu, lost<L>(c, n))) {
            c = cw = c_in;
            if (R > 1) {
#pragma unroll 1
                for (int k = R - 1; k >= 0; --k) {
                    if (k == at.rank) cw = c;
                    c = fold_any<L>(c, meet.total[b][0][k][lane], meet.total[b][1][k][lane]);
                }
            }
            V x = cw;
#pragma unroll 1
            for (int w = kWarps - 1; w >= 0; --w) {
                if (w == warp) cw = x;
                x = fold_any<L>(x, meet.warp[0][0][w][lane], meet.warp[0][2][w][lane]);
            }
            if (R == 1) c = x;
            if (LW == 16 && lane < 16) cw = fold_any<L>(cw, c1, e1);
            second(std::false_type{});
        }
        if (A == kTma) fence_async_smem();  // the gates put there come before the next tiles
        __syncthreads();  // every warp is done with the tiles and the meeting
        if (walk.issuer() && s + kStages < steps) walk.load(s + kStages, chunk_of(s + kStages));
        walk.copy_rows(s + kStages, chunk_of(s + kStages));
        __syncwarp();
    }
    walk.end();
    for (int k = steps * R + at.rank; k * Cut<LW>::kTokens < p.n_tok; k += R) {  // past the sequence's end
        const int t0 = k * Cut<LW>::kTokens + at.run * kTok;
        blank<T, A>(static_cast<T*>(p.dg) + (int64_t)at.seq * p.seq_dg + at.c0, p.s_dg, t0, p.n_tok, n);
        blank<T, A>(static_cast<T*>(p.dv) + (int64_t)at.seq * p.seq_dv + at.c0, p.s_dv, t0, p.n_tok, n);
    }
    if (p.dh0 && at.rank == 0 && warp == 0 && lane < LW) st_state<L>(p.dh0 + (int64_t)at.seq * p.seq_dh0 + at.c0, n, c);
}

// A step of a lane's channels, one by one.
template <typename L, bool kAny>
__device__ __forceinline__ void move(typename L::V c, float (&h)[L::kN], typename L::V v) {
    float x[L::kN], y[L::kN];
    L::to(c, x), L::to(v, y);
#pragma unroll
    for (int e = 0; e < L::kN; ++e) h[e] = kAny ? moved_any(x[e], h[e], y[e]) : moved(x[e], h[e], y[e]);
}

// Up to NT tokens: a warp has the channels of one slab of one sequence.
template <typename T, Access A, bool GRAD, int NT>
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

    V w[NT];
    uint32_t gw[NT], vw[NT], yw[GRAD ? NT : 1];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        const bool live = i < len;
        gw[i] = live ? ld_raw<T, A>(g + i * p.s_g, n) : L::kInf;
        vw[i] = live ? ld_raw<T, A>(v + i * p.s_v, n) : 0u;
        if constexpr (GRAD) yw[i] = live ? ld_raw<T, A>(dy + i * p.s_dy, n) : 0u;
    }
#pragma unroll
    for (int i = 0; i < NT; ++i) w[i] = gate_decay<T>(L::unpack(gw[i]));
    if constexpr (!GRAD) {
        T* y = static_cast<T*>(p.y) + (int64_t)seq * p.seq_y + c0;
        const V h0 = ld_state<L>(p.h0 ? p.h0 + (int64_t)seq * p.seq_h0 + c0 : nullptr, n);
        float h[N];
        L::to(h0, h);
        if (p.states && p.n_tok > 0) st_state<L>(p.states + (int64_t)seq * p.n_chan + c0, n, h0);
        uint32_t out[NT];
#pragma unroll
        for (int i = 0; i < NT; ++i) {  // past the end z is 0
            move<L, false>(w[i], h, L::unpack(vw[i]));
            out[i] = i < len ? L::pack(L::of(h)) : 0u;
        }
        // no step makes an infinity or a NaN finite again
        if (!finite(h[0]) || !finite(h[N - 1])) {
            L::to(h0, h);
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                move<L, true>(w[i], h, L::unpack(vw[i]));
                out[i] = i < len ? L::pack(L::of(h)) : 0u;
            }
        }
#pragma unroll
        for (int i = 0; i < NT; ++i)
            if (i < p.n_tok) st_raw<T, A>(y + i * p.s_y, n, out[i]);
        st_state<L>(p.h1 + (int64_t)seq * p.seq_h1 + c0, n, L::of(h));
    } else {
        T* dg = static_cast<T*>(p.dg) + (int64_t)seq * p.seq_dg + c0;
        T* dv = static_cast<T*>(p.dv) + (int64_t)seq * p.seq_dv + c0;
        float h[N], c[N];
        L::to(ld_state<L>(p.n_tok > 0 ? p.states + (int64_t)seq * p.n_chan + c0 : nullptr, n), h);
        L::to(ld_state<L>(p.dh1 ? p.dh1 + (int64_t)seq * p.seq_dh1 + c0 : nullptr, n), c);
        V q[NT];
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            float x[N], v_[N];
            L::to(w[i], x), L::to(L::unpack(vw[i]), v_);
#pragma unroll
            for (int e = 0; e < N; ++e) x[e] = slope(x[e]) * (h[e] - v_[e]);
            q[i] = L::of(x);
            move<L, true>(w[i], h, L::unpack(vw[i]));
        }
#pragma unroll
        for (int i = NT - 1; i >= 0; --i) {
            if (i >= p.n_tok) continue;
            const bool live = i < len;
            float x[N], y_[N], lam[N], take[N];
            L::to(w[i], x), L::to(L::unpack(yw[i]), y_);
#pragma unroll
            for (int e = 0; e < N; ++e) {
                lam[e] = y_[e] + c[e];
                take[e] = taken(x[e], lam[e]);
                c[e] = kept(x[e], lam[e]);
            }
            st_raw<T, A>(dg + i * p.s_dg, n, live ? L::pack(L::mul(L::of(lam), q[i])) : 0u);
            st_raw<T, A>(dv + i * p.s_dv, n, live ? L::pack(L::of(take)) : 0u);
        }
        if (p.dh0) st_state<L>(p.dh0 + (int64_t)seq * p.seq_dh0 + c0, n, L::of(c));
    }
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------
// Steps of tiles, and of copied rows, that fit beside two CTAs per SM.
constexpr int kFwdStages = 3, kGradStages = 2;
constexpr int kRowStages = 2, kGradRowStages = 1;
constexpr size_t tiles_smem(int tensors, int stages) { return (size_t)stages * tensors * kTileBytes + 128; }
// The gradient's rows have their gates beside them, 8 bytes for 4 of a tile.
template <int LW>
constexpr size_t rows_smem(int tensors, int stages) {
    return (size_t)stages * tensors * Cut<LW>::kRowTile + (tensors == 3 ? 2 * kTileBytes : 0) + 128;
}

// [n_seq][n_tok][n_chan] in boxes of row_bytes bytes of a tile's tokens; false when TMA
// cannot describe it.  Rows and channels past the ends read as zero.
bool make_map_tok(const helix_ctx* ctx, CUtensorMap* m, const GatedParams& p, const void* base, int64_t s_tok,
                  int64_t s_seq, int size, int row_bytes) {
    if (reinterpret_cast<uintptr_t>(base) % 16) return false;
    const int64_t row = ((int64_t)p.n_chan * size + 15) / 16 * 16;
    const int64_t bt = p.n_tok > 1 ? s_tok * size : row, bs = p.n_seq > 1 ? s_seq * size : row;
    if (bt <= 0 || bs <= 0 || bt % 16 || bs % 16) return false;
    const auto fn = reinterpret_cast<tc::EncodeFn>(ctx->encode_tiled);
    cuuint64_t dims[3] = {(cuuint64_t)p.n_chan, (cuuint64_t)p.n_tok, (cuuint64_t)p.n_seq};
    cuuint64_t strides[2] = {(cuuint64_t)bt, (cuuint64_t)bs};
    cuuint32_t box[3] = {(cuuint32_t)(row_bytes / size), (cuuint32_t)(kTileBytes / row_bytes), 1};
    cuuint32_t es[3] = {1, 1, 1};
    return fn(m, size == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
              const_cast<void*>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool make_maps(const helix_ctx* ctx, GatedMaps* m, const GatedParams& p, bool grad, int size, int row_bytes) {
    std::memset(m, 0, sizeof(*m));
    if (!ctx->encode_tiled || p.n_tok <= 0) return false;
    if (!make_map_tok(ctx, &m->in[0], p, p.g, p.s_g, p.seq_g, size, row_bytes)) return false;
    if (!make_map_tok(ctx, &m->in[1], p, p.v, p.s_v, p.seq_v, size, row_bytes)) return false;
    return !grad || make_map_tok(ctx, &m->in[2], p, p.dy, p.s_dy, p.seq_dy, size, row_bytes);
}

// Lanes of a row and CTAs of a cluster: the choice with the fewest steps,
// counting the waves that its clusters take, two CTAs per SM (large clusters
// leave SMs of a GPC idle), and two steps to fill and drain each.  Narrow rows
// serve few channels: 1 x 131072 x 1024 bf16 takes 193 us with
// them, 310 without.  Clusters of 8 take those 193 us, of 4 215, of 2 404, one
// CTA 672; at 4 x 8192 x 2048 one takes 78 us, two 79, four 85, eight 99.
struct GatedCut {
    int lanes = 32, cluster = 1;
};
GatedCut cut_of(const helix_ctx* ctx, const GatedParams& p, int lane_channels) {
    GatedCut best;
    int64_t least = INT64_MAX;
    for (int lanes = 32; lanes >= 16; lanes /= 2) {
        const int64_t cb = lanes * lane_channels, groups = (int64_t)p.n_seq * ((p.n_chan + cb - 1) / cb);
        const int64_t tokens = kChunk * (32 / lanes), chunks = (p.n_tok + tokens - 1) / tokens;
        for (int i = 0, r = 1; r <= kMaxCluster; ++i, r *= 2) {
            const int64_t at_once = ctx->gated_clusters[i];
            if (at_once <= 0 || (r > 1 && r >= 2 * chunks)) continue;
            const int64_t cost = (groups + at_once - 1) / at_once * ((chunks + r - 1) / r + 2);
            if (cost < least) {
                least = cost;
                best.lanes = lanes, best.cluster = r;
            }
        }
    }
    return best;
}

struct ClusterLaunch {
    cudaLaunchConfig_t  cfg{};
    cudaLaunchAttribute at{};
    ClusterLaunch(int64_t grid, int cluster, size_t smem, void* stream) {
        cfg.gridDim = dim3((unsigned)grid);
        cfg.blockDim = dim3((unsigned)kThreads);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = static_cast<cudaStream_t>(stream);
        at.id = cudaLaunchAttributeClusterDimension;
        at.val.clusterDim.x = (unsigned)cluster;
        at.val.clusterDim.y = at.val.clusterDim.z = 1;
        cfg.attrs = &at;
        cfg.numAttrs = 1;
    }
};

template <typename T, Access A, int NT>
int launch_few(const GatedParams& p, int64_t groups, bool grad, void* stream) {
    const dim3 grid((unsigned)((groups + kFewWarps - 1) / kFewWarps)), block(32 * kFewWarps);
    return grad ? block_launch(gated_few_kernel<T, A, true, NT>, grid, block, 0, stream, p)
                : block_launch(gated_few_kernel<T, A, false, NT>, grid, block, 0, stream, p);
}

template <typename T, Access A, int LW>
int launch_gated_a(const GatedMaps& maps, GatedParams p, const GatedCut& cut, bool grad, void* stream) {
    constexpr int CB = LW * Lane<T>::kN;
    const int64_t groups = (int64_t)p.n_seq * ((p.n_chan + CB - 1) / CB);
    p.cluster = cut.cluster;
    const int64_t grid = groups * p.cluster;
    if (grad) {
        ClusterLaunch l(grid, p.cluster, A == kTma ? tiles_smem(3, kGradStages) : rows_smem<LW>(3, kGradRowStages),
                        stream);
        return cudaLaunchKernelEx(&l.cfg, gated_grad_kernel<T, A, A == kTma ? kGradStages : kGradRowStages, LW>, maps,
                                  p);
    }
    ClusterLaunch l(grid, p.cluster, A == kTma ? tiles_smem(2, kFwdStages) : rows_smem<LW>(2, kRowStages), stream);
    return cudaLaunchKernelEx(&l.cfg, gated_kernel<T, A, A == kTma ? kFwdStages : kRowStages, LW>, maps, p);
}

template <typename T, Access A>
int launch_gated_few(const GatedParams& p, bool grad, void* stream) {
    constexpr int CB = 32 * Lane<T>::kN;
    const int64_t groups = (int64_t)p.n_seq * ((p.n_chan + CB - 1) / CB);
    return p.n_tok <= 1   ? launch_few<T, A, 1>(p, groups, grad, stream)
           : p.n_tok <= 4 ? launch_few<T, A, 4>(p, groups, grad, stream)
                          : launch_few<T, A, kTok>(p, groups, grad, stream);
}

bool whole_lines(const GatedParams& p, bool grad, int64_t size) {
    auto lines = [&](const void* at, int64_t s_tok, int64_t s_seq) {
        return reinterpret_cast<uintptr_t>(at) % 128 == 0 && s_tok * size % 128 == 0 &&
               (p.n_seq <= 1 || s_seq * size % 128 == 0);
    };
    return lines(p.v, p.s_v, p.seq_v) && lines(p.g, p.s_g, p.seq_g) && (!grad || lines(p.dy, p.s_dy, p.seq_dy));
}

template <typename T>
int launch_gated_t(const helix_ctx* ctx, const GatedParams& p, bool word, bool grad, void* stream) {
    constexpr int N = Lane<T>::kN;
    if (p.n_tok <= kTok) {
        if constexpr (N == 2)
            if (!word) return launch_gated_few<T, kHalf>(p, grad, stream);
        return launch_gated_few<T, kWord>(p, grad, stream);
    }
    const GatedCut cut = cut_of(ctx, p, N);
    // Outputs are stored a word at a time in the TMA form too.  Rows of f32
    // that do not start at lines of 128 bytes are read faster as rows (4 x 8192
    // x 2040: 143 us against 203, gradient 306 against 358; bf16 118 against 93),
    // unless the cut is narrow.
    if (word && (N == 2 || cut.lanes == 16 || whole_lines(p, grad, sizeof(T)))) {
        GatedMaps maps;
        if (make_maps(ctx, &maps, p, grad, sizeof(T), 4 * cut.lanes))
            return cut.lanes == 16 ? launch_gated_a<T, kTma, 16>(maps, p, cut, grad, stream)
                                   : launch_gated_a<T, kTma, 32>(maps, p, cut, grad, stream);
    }
    GatedMaps none;
    std::memset(&none, 0, sizeof(none));
    if constexpr (N == 2)
        if (!word)
            return cut.lanes == 16 ? launch_gated_a<T, kHalf, 16>(none, p, cut, grad, stream)
                                   : launch_gated_a<T, kHalf, 32>(none, p, cut, grad, stream);
    return cut.lanes == 16 ? launch_gated_a<T, kWord, 16>(none, p, cut, grad, stream)
                           : launch_gated_a<T, kWord, 32>(none, p, cut, grad, stream);
}

int launch_gated_any(const helix_ctx* ctx, const helix_gated_scan_desc& d, const GatedParams& p, bool word, bool grad,
                     void* stream) {
    return d.io_dtype == HELIX_F32 ? launch_gated_t<float>(ctx, p, word, grad, stream)
                                   : launch_gated_t<__nv_bfloat16>(ctx, p, word, grad, stream);
}

template <typename K>
int set_smem(K kernel, size_t bytes) {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
}

template <typename T, int LW>
int configure_tiles() {
    const int e = set_smem(gated_kernel<T, kTma, kFwdStages, LW>, tiles_smem(2, kFwdStages));
    return e != cudaSuccess ? e : set_smem(gated_grad_kernel<T, kTma, kGradStages, LW>, tiles_smem(3, kGradStages));
}
template <typename T, Access A, int LW>
int configure_rows() {
    const int e = set_smem(gated_kernel<T, A, kRowStages, LW>, rows_smem<LW>(2, kRowStages));
    if (e != cudaSuccess) return e;
    return set_smem(gated_grad_kernel<T, A, kGradRowStages, LW>, rows_smem<LW>(3, kGradRowStages));
}

}  // namespace

int configure_gated(helix_ctx* ctx) {
    int e;
    if ((e = configure_tiles<float, 32>()) != cudaSuccess) return e;
    if ((e = configure_tiles<float, 16>()) != cudaSuccess) return e;
    if ((e = configure_tiles<__nv_bfloat16, 32>()) != cudaSuccess) return e;
    if ((e = configure_tiles<__nv_bfloat16, 16>()) != cudaSuccess) return e;
    if ((e = configure_rows<float, kWord, 32>()) != cudaSuccess) return e;
    if ((e = configure_rows<float, kWord, 16>()) != cudaSuccess) return e;
    if ((e = configure_rows<__nv_bfloat16, kWord, 32>()) != cudaSuccess) return e;
    if ((e = configure_rows<__nv_bfloat16, kWord, 16>()) != cudaSuccess) return e;
    if ((e = configure_rows<__nv_bfloat16, kHalf, 32>()) != cudaSuccess) return e;
    if ((e = configure_rows<__nv_bfloat16, kHalf, 16>()) != cudaSuccess) return e;
    for (int i = 0, r = 1; r <= kMaxCluster; ++i, r *= 2) {
        ClusterLaunch l(r, r, tiles_smem(2, kFwdStages), nullptr);
        e = cudaOccupancyMaxActiveClusters(&ctx->gated_clusters[i], gated_kernel<__nv_bfloat16, kTma, kFwdStages, 32>,
                                           &l.cfg);
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
