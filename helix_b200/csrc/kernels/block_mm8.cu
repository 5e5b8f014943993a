// block_mm8.cu -- product of e4m3 matrices with an fp32 scale for each block
// of 128 along k, on tcgen05.
//
//     out[i][j] = sum_b sa[i][b] sb[j][b] D_b[i][j],  D_b = sum_{k in b} a[i][k] b[j][k]
//
// The scales differ from block to block of k, so the sum over blocks cannot
// stay in the tensor core's accumulator: each block's D_b is four MMAs of
// K = 32 into one of several TMEM buffers, and the epilogue warps add
// (sa sb) D_b to fp32 registers while the next blocks' MMAs run.
//
// A CTA has a tile of 128 rows of P x BN rows of Q: warp 0 issues the TMA
// loads (128-byte rows, one block of k per stage), warps 1 and 2 the MMAs of
// the even and the odd blocks, warps 3-10 are the epilogue, four of them (one
// for each quarter of the rows, the TMEM lanes that a warp can reach) for the
// even blocks and four for the odd ones.  A block's hand-offs take a thread
// longer than its MMAs take the tensor core, so each has two blocks' time.  P
// is a and Q is b, or the other way round where a has few rows: the MMA is
// always 128 rows tall, so the weight takes those and the tokens become a
// narrow N.
//
// With few tiles the blocks of k are shared by a cluster of CTAs.  The partial
// sums (of even and odd blocks, of all CTAs) meet in (distributed) shared
// memory, and every CTA adds up and writes a share of the columns, in the
// order of the ranks.
//
// Measured (this kernel; that of large products below): 16 x 8192 x 4096 8.2 us,
// 128 x 8192 x 4096 13.4; the weight's bytes take 5.2 at the measured copy rate.
// The rest is the chain of one CTA's work: launch, first loads, the last block's
// hand-offs and the meeting of the cluster, with 16 blocks of k in between.
//
// Every wait is bounded: one that runs out records kFaultProduct, the CTA
// lets its copies and MMAs land, frees its TMEM and returns.
#include <cooperative_groups.h>

#include <algorithm>
#include <cstring>

#include "block_common.cuh"
#include "common.cuh"
#include "tc_shared.cuh"

namespace hx {
namespace {

namespace cg = cooperative_groups;
using namespace umma;

constexpr int kRows = 128;                 // of P in a tile
constexpr int kBk = HELIX_GROUP;           // bytes of k in a stage: one scale block
constexpr int kEpiWarps = 8;
constexpr int kMmThreads = 32 * (3 + kEpiWarps);

template <int BN>
struct Mm8Cfg {
    static constexpr int kStageBytes = (kRows + BN) * kBk;
    static constexpr int kStages = BN == 64 ? 8 : BN == 32 ? 5 : 6;
    static constexpr int kPerSm = BN == 64 ? 1 : 2;          // CTAs that fit
    static constexpr int kBufs = 4;                          // TMEM accumulators
    static constexpr int kCols = kBufs * BN;
    static constexpr int kLoad = BN < 32 ? BN : 32;          // columns read at once
    static constexpr int kPiece = 16;                        // blocks of k whose column scales are staged at once
    static constexpr size_t kSmem = (size_t)kStages * kStageBytes + 1024;
    static_assert(2 * BN * kRows * sizeof(float) <= (size_t)kStages * kStageBytes, "partial sums");
};

struct Mm8Maps {
    CUtensorMap p, q;
};

// A place in a ring of N barriers, and the parity of its turn.
template <int N>
struct Ring {
    int      at = 0;
    uint32_t parity = 0;
    __device__ __forceinline__ void next() {
        if (++at == N) at = 0, parity ^= 1u;
    }
};

// Whether the phase is over, without waiting for it.
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}

// The first n of v: consecutive columns qc.. of row pr of P.
template <typename T>
__device__ __forceinline__ void st_out(const Mm8Params& a, int pr, int qc, int n, const float (&v)[8]) {
    if (pr >= a.p.rows) return;
    if (a.swap) {  // out[q][p]: lanes hold consecutive p
        T* o = static_cast<T*>(a.out) + (int64_t)qc * a.ld_out + pr;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n && qc + i < a.q.rows) o[(int64_t)i * a.ld_out] = from_f32<T>(v[i]);
        return;
    }
    T* o = static_cast<T*>(a.out) + (int64_t)pr * a.ld_out + qc;
    if (n == 8 && a.vec_out && qc + 8 <= a.q.rows) {
        st8(o, v);
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < n && qc + i < a.q.rows) o[i] = from_f32<T>(v[i]);
}

template <int BN, bool QROWS, typename T>
__global__ void __launch_bounds__(kMmThreads, Mm8Cfg<BN>::kPerSm) mm8_kernel(const __grid_constant__ Mm8Maps maps,
                                                                             const __grid_constant__ Mm8Params a) {
    using Cfg = Mm8Cfg<BN>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = tc::align1024(smem_raw);
    __shared__ uint64_t full[Cfg::kStages], empty[Cfg::kStages], acc_full[Cfg::kBufs], acc_empty[Cfg::kBufs], drain[2];
    __shared__ uint32_t tmem_slot;
    __shared__ __align__(16) float col_scale[QROWS ? Cfg::kPiece : 1][QROWS ? BN : 4];

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)(blockIdx.x % (unsigned)a.splits), tile = (int)(blockIdx.x / (unsigned)a.splits);
    const int p0 = tile / a.tiles_q * kRows, q0 = tile % a.tiles_q * BN;
    const int kb0 = (int)((int64_t)a.k_blocks * rank / a.splits);
    const int nkb = (int)((int64_t)a.k_blocks * (rank + 1) / a.splits) - kb0;

    auto load = [&](int i, int s) {
        uint8_t* st = smem + s * Cfg::kStageBytes;
        mbar_expect_tx(&full[s], Cfg::kStageBytes);
        tma_load_2d(st, &maps.p, &full[s], (kb0 + i) * kBk, p0);
        tma_load_2d(st + kRows * kBk, &maps.q, &full[s], (kb0 + i) * kBk, q0);
    };
    if (threadIdx.x == 0) {
#pragma unroll
        for (int i = 0; i < Cfg::kStages; ++i) mbar_init(&full[i], 1), mbar_init(&empty[i], 1);
#pragma unroll
        for (int i = 0; i < Cfg::kBufs; ++i) mbar_init(&acc_full[i], 1), mbar_init(&acc_empty[i], kEpiWarps / 2);
        mbar_init(&drain[0], 1), mbar_init(&drain[1], 1);
        fence_mbar_init();
        // the first loads wait for nobody
        for (int i = 0; i < Cfg::kStages && i < nkb; ++i) load(i, i);
    }
    __syncwarp();
    if (warp == 1) tmem_alloc(&tmem_slot, Cfg::kCols);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;

    auto wait = [&](uint64_t* bar, uint32_t parity) {
        if (mbar_wait(bar, parity, tc::kWaitBudget)) return true;
        if (a.fault) atomicCAS(a.fault, 0u, (unsigned)kFaultProduct);
        return false;
    };

    const int group = (warp - 3) / 4;                 // of an epilogue warp: 0 even blocks, 1 odd
    const int row = 32 * (warp & 3) + lane;           // its TMEM lane
    float acc[BN];
#pragma unroll
    for (int i = 0; i < BN; ++i) acc[i] = 0.0f;

    if (warp == 0) {
        if (lane == 0) {
            Ring<Cfg::kStages> st;
            int i = min(Cfg::kStages, nkb);
            for (; i < nkb; ++i) {
                if (!wait(&empty[st.at], st.parity)) break;
                load(i, st.at);
                st.next();
            }
            // whatever the other warps do, the loads issued land before the CTA ends
            for (int j = i > Cfg::kStages ? i - Cfg::kStages : 0; j < i; ++j)
                mbar_wait(&full[j % Cfg::kStages], (uint32_t)((j / Cfg::kStages) & 1), tc::kWaitBudget);
        }
    } else if (warp < 3) {
        if (lane == 0) {
            constexpr uint32_t idesc = idesc_e4m3(kRows, BN);
            const uint32_t base = smem_u32(smem);
            const int first = warp - 1;
            Ring<Cfg::kStages> st;
            Ring<Cfg::kBufs> buf;
            if (first) st.next(), buf.next();
            // A wait costs its latency even when nothing is left to wait for;
            // the next block's two are polled between its issue and its commits.
            bool ready = false, free = true;
            int i = first;
            for (; i < nkb; i += 2) {
                if (!free && !wait(&acc_empty[buf.at], buf.parity ^ 1u)) break;
                if (!ready && !wait(&full[st.at], st.parity)) break;
                tc_fence_after();
                const uint32_t from = base + st.at * Cfg::kStageBytes;
                const uint64_t dp = sdesc_sw128(from, 16, 1024), dq = sdesc_sw128(from + kRows * kBk, 16, 1024);
#pragma unroll
                for (int ks = 0; ks < 4; ++ks)
                    mma_e4m3(tmem + buf.at * BN, tc::desc_add(dp, 32 * ks), tc::desc_add(dq, 32 * ks), idesc, ks > 0);
                uint64_t *done = &acc_full[buf.at], *read = &empty[st.at];
                st.next(), st.next();
                buf.next(), buf.next();
                ready = i + 2 < nkb && mbar_try_wait(&full[st.at], st.parity);
                free = i + 2 < Cfg::kBufs || mbar_try_wait(&acc_empty[buf.at], buf.parity ^ 1u);
                mma_commit(done);
                mma_commit(read);
            }
            if (i < nkb) {
                mma_commit(&drain[first]);
                mbar_wait(&drain[first], 0, tc::kWaitBudget);
            }
        }
    } else {
        const int tid = threadIdx.x - 96;             // 0 .. 255
        const uint32_t lane_addr = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
        // the row's scale one of the group's blocks ahead; the columns', where
        // they share one, too
        const float* ps = a.p.scale + (int64_t)(min(p0 + row, a.p.rows - 1) / a.p.per) * a.p.ld_scale + kb0;
        const float* qs = a.q.scale + (int64_t)(min(q0, a.q.rows - 1) / a.q.per) * a.q.ld_scale + kb0;
        float ps_next = __ldg(ps + min(group, nkb - 1)), ps_then = __ldg(ps + min(group + 2, nkb - 1));
        float qs_next = 1.0f, qs_then = 1.0f;
        if (!QROWS) qs_next = __ldg(qs + min(group, nkb - 1)), qs_then = __ldg(qs + min(group + 2, nkb - 1));
        // column scales of kPiece blocks: value j of the piece at i is block
        // i + j % kPiece of column j / kPiece
        constexpr int kMine = (BN * Cfg::kPiece + 32 * kEpiWarps - 1) / (32 * kEpiWarps);
        float piece[QROWS ? kMine : 1];
        auto fetch = [&](int i) {
            if constexpr (QROWS) {
#pragma unroll
                for (int j = 0; j < kMine; ++j) {
                    const int e = tid + 32 * kEpiWarps * j, q = min(q0 + e / Cfg::kPiece, a.q.rows - 1);
                    piece[j] = __ldg(a.q.scale + (int64_t)q * a.q.ld_scale + kb0 + min(i + e % Cfg::kPiece, nkb - 1));
                }
            }
        };
        fetch(0);
        Ring<Cfg::kBufs> buf;
        if (group) buf.next();
        bool alive = true;  // once a wait has run out no other is waited for, and the rest is garbage
        for (int i0 = 0; i0 < nkb; i0 += Cfg::kPiece) {
            if constexpr (QROWS) {
                named_sync(1, 32 * kEpiWarps);  // the last piece is read
#pragma unroll
                for (int j = 0; j < kMine; ++j) {
                    const int e = tid + 32 * kEpiWarps * j;
                    if (e < BN * Cfg::kPiece) col_scale[e % Cfg::kPiece][e / Cfg::kPiece] = piece[j];
                }
                named_sync(1, 32 * kEpiWarps);
                if (i0 + Cfg::kPiece < nkb) fetch(i0 + Cfg::kPiece);
            }
            for (int i = i0 + group; i < nkb && i < i0 + Cfg::kPiece; i += 2) {
                const float r = QROWS ? ps_next : ps_next * qs_next;
                ps_next = ps_then;
                ps_then = __ldg(ps + min(i + 4, nkb - 1));
                if constexpr (!QROWS) {
                    qs_next = qs_then;
                    qs_then = __ldg(qs + min(i + 4, nkb - 1));
                }
                if (alive) alive = __all_sync(0xffffffffu, wait(&acc_full[buf.at], buf.parity));
                tc_fence_after();
#pragma unroll
                for (int c = 0; c < BN; c += Cfg::kLoad) {
                    uint32_t v[Cfg::kLoad];
                    tmem_ld(lane_addr + buf.at * BN + c, v);
                    tmem_wait_ld(v);
                    if (c + Cfg::kLoad == BN) {  // all read
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&acc_empty[buf.at]);
                    }
#pragma unroll
                    for (int e = 0; e < Cfg::kLoad; ++e) {
                        const float s = QROWS ? r * col_scale[i % Cfg::kPiece][c + e] : r;
                        acc[c + e] = fmaf(__uint_as_float(v[e]), s, acc[c + e]);
                    }
                }
                buf.next(), buf.next();
            }
        }
    }

    // every load and MMA of this CTA has retired, so the stages are free
    __syncthreads();
    float* part = reinterpret_cast<float*>(smem);  // [2][BN][128]
    if (warp >= 3) {
#pragma unroll
        for (int c = 0; c < BN; ++c) part[(group * BN + c) * kRows + row] = acc[c];
    }
    cg::cluster_group cluster = cg::this_cluster();
    if (a.splits > 1)
        cluster.sync();
    else
        __syncthreads();
    if (warp >= 3) {
        const int run = BN / 2 / a.splits;  // columns of this thread's share
        const int c0 = rank * (BN / a.splits) + group * run;
        for (int c = 0; c < run; c += 8) {
            const int n = min(8, run - c);
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = 0.0f;
            for (int k = 0; k < a.splits; ++k) {
                const float* from = a.splits > 1 ? cluster.map_shared_rank(part, k) : part;
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (e < n) v[e] += from[(c0 + c + e) * kRows + row] + from[(BN + c0 + c + e) * kRows + row];
            }
            st_out<T>(a, p0 + row, q0 + c0 + c, n, v);
        }
    }
    if (a.splits > 1) cluster.sync();  // a peer may still be reading this CTA's share
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_relinquish();
        tmem_dealloc(tmem, Cfg::kCols);
    }
}

// ---------------------------------------------------------------------------
// Large products: pairs of CTAs, tiles of 256 x BN.
//
// One CTA's MMA reads 128 + BN rows of shared memory per block; the pair's
// MMA (cta_group::2) lets each CTA hold half of the columns' operand, so a
// tile of 256 x 256 moves as many bytes per CTA as one of 128 x 128 for four
// times the products, half of them each.  The grid is persistent, one CTA per
// SM: the blocks of k of all of a pair's tiles run through one pipeline of
// stages and TMEM buffers, and the next tile's MMAs run while the epilogue
// writes.  An epilogue warp has 32 rows and half of the columns; it stages its
// part in shared memory of its own and stores it by TMA.
//
// Where b's scales go by blocks of 128, an accumulator of one row per lane needs
// one scale per block of k.  Where they go by rows every column has its own:
// with a row per lane, a lane would read all of them from shared memory (64
// 8-byte reads per block of k); with the fragments of 16 lanes x 8 columns it has
// 4 rows, and a quarter of the columns.  There the epilogue is also what the
// MMAs wait for (two multiply-adds a value and block, not one), so a block's
// first TMEM read is issued before the last block's sums are done, if its MMAs
// are (8192 x 8192 x 4096 to f32: 414 -> 376 us; by blocks, where the epilogue
// waits for the MMAs, 264 -> 278, so not there).
//
// Measured: 8192 x 8192 x 4096 bf16 258 us, 2.1 PFLOP/s, 64 % of twice the
// measured bf16 rate; by rows to f32 352 us.  Bound by the tensor core and the
// hand-offs between it and the epilogue (a block's sum has to leave TMEM before
// its buffer is free, and there are two), by rows by the epilogue's arithmetic.
// ---------------------------------------------------------------------------
// Warp 0 issues the loads, 1 and 2 the MMAs of every other block of k (a
// block's waits, four MMAs and commits take one thread 750 cycles, three times
// what the MMAs themselves take at BN = 128), 3 stages scales, 4-11 are
// the epilogue: 32 rows and half of the columns each.  The first warpgroup hands registers to
// the others, whose accumulators take up to 128 each: 128 x 40 + 256 x 232 (or
// 72 and 216, when warp 3 has work) = 384 x 168, the registers that the block
// is launched with.
constexpr int kPairThreads = 32 * (4 + kEpiWarps);

template <int BN, bool QROWS>
struct PairCfg {
    static constexpr int kStageBytes = (kRows + BN / 2) * kBk;   // per CTA
    static constexpr int kStages = BN == 256 ? 5 : 6;
    static constexpr int kOuts = QROWS ? 1 : 2;                  // stagings of an epilogue warp
    static constexpr int kBufs = 512 / BN;
    static constexpr int kRun = BN / 2;                          // columns of an epilogue warp
    static constexpr int kPiece = 8;                             // blocks of k whose scales are staged at once
    static_assert(kPiece == 8, "two quads");
    static constexpr int kOutBytes = 32 * 128;                   // of one
    static constexpr size_t kSmem = (size_t)kStages * kStageBytes + kEpiWarps * kOuts * kOutBytes + 1024;
};

struct PairMaps {
    CUtensorMap p, q, out;
};

// Tiles in strips of 8 tile rows, down the strip first: the tiles in flight
// share rows of both operands in L2.
__device__ __forceinline__ void pair_tile(int tile, int tiles_p, int tiles_q, int* tp, int* tq) {
    constexpr int kStrip = 8;
    const int strip = tile / (kStrip * tiles_q), first = strip * kStrip;
    const int high = min(kStrip, tiles_p - first), in = tile - first * tiles_q;
    *tp = first + in % high;
    *tq = in / high;
}

template <int BN, bool QROWS, typename T>
__global__ void __launch_bounds__(kPairThreads, 1)
    mm8_pair_kernel(const __grid_constant__ PairMaps maps, const __grid_constant__ Mm8Params a) {
    using Cfg = PairCfg<BN, QROWS>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = tc::align1024(smem_raw);
    __shared__ uint64_t full[Cfg::kStages], empty[Cfg::kStages], acc_full[Cfg::kBufs], acc_empty[Cfg::kBufs], drain[2];
    __shared__ uint64_t sc_full[2], sc_empty[2];
    __shared__ uint32_t tmem_slot;
    __shared__ __align__(16) float row_scale[2][QROWS ? Cfg::kPiece : 1][QROWS ? kRows : 4];
    __shared__ __align__(16) float col_scale[2][QROWS ? Cfg::kPiece : 1][QROWS ? BN : 4];

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)(blockIdx.x & 1u), pair = (int)(blockIdx.x >> 1), pairs = (int)(gridDim.x >> 1);
    const int tiles_p = (a.p.rows + 2 * kRows - 1) / (2 * kRows), n_tiles = tiles_p * a.tiles_q;
    const int nkb = a.k_blocks;

    if (threadIdx.x == 0) {
        prefetch_tmap(&maps.p);
        prefetch_tmap(&maps.q);
#pragma unroll
        for (int i = 0; i < Cfg::kStages; ++i) mbar_init(&full[i], 1), mbar_init(&empty[i], 1);
#pragma unroll
        for (int i = 0; i < Cfg::kBufs; ++i) mbar_init(&acc_full[i], 1), mbar_init(&acc_empty[i], 2 * kEpiWarps);
#pragma unroll
        for (int i = 0; i < 2; ++i) mbar_init(&sc_full[i], 1), mbar_init(&sc_empty[i], kEpiWarps);
        mbar_init(&drain[0], 1), mbar_init(&drain[1], 1);
        fence_mbar_init();
    }
    if (warp == 1) tmem_alloc_pair(&tmem_slot, 512);
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();  // both CTAs' barriers and TMEM stand
    tc_fence_after();
    const uint32_t tmem = tmem_slot;

    auto wait = [&](uint64_t* bar, uint32_t parity) {
        if (mbar_wait(bar, parity, tc::kWaitBudget)) return true;
        if (a.fault) atomicCAS(a.fault, 0u, (unsigned)kFaultProduct);
        return false;
    };

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(QROWS ? 72 : 40));
        if (warp == 0 && lane == 0) {
            Ring<Cfg::kStages> st;  // runs over the blocks of k of all tiles
            int issued = 0;
            bool ok = true;
            for (int tile = pair; ok && tile < n_tiles; tile += pairs) {
                int tp, tq;
                pair_tile(tile, tiles_p, a.tiles_q, &tp, &tq);
                const int row_p = (2 * tp + rank) * kRows, row_q = tq * BN + rank * (BN / 2);
                for (int kb = 0; kb < nkb; ++kb) {
                    if (issued >= Cfg::kStages && !(ok = wait(&empty[st.at], st.parity ^ 1u))) break;
                    uint8_t* to = smem + st.at * Cfg::kStageBytes;
                    // the even CTA's barrier counts both CTAs' bytes
                    if (rank == 0) mbar_expect_tx(&full[st.at], 2 * Cfg::kStageBytes);
                    const uint32_t bar = cluster_addr(&full[st.at], 0);
                    tma_load_2d_pair(to, &maps.p, bar, kb * kBk, row_p);
                    tma_load_2d_pair(to + kRows * kBk, &maps.q, bar, kb * kBk, row_q);
                    st.next();
                    ++issued;
                }
            }
            // the loads issued land before the pair ends
            if (rank == 0)
                for (int j = issued > Cfg::kStages ? issued - Cfg::kStages : 0; j < issued; ++j)
                    mbar_wait(&full[j % Cfg::kStages], (uint32_t)((j / Cfg::kStages) & 1), tc::kWaitBudget);
        } else if (warp < 3 && lane == 0 && rank == 0) {
            constexpr uint32_t idesc = idesc_e4m3(2 * kRows, BN);
            const uint32_t base = smem_u32(smem);
            const int mine = pair < n_tiles ? (n_tiles - pair + pairs - 1) / pairs : 0;
            const int total = mine * nkb, first = warp - 1;
            Ring<Cfg::kStages> st;
            Ring<Cfg::kBufs> buf;
            if (first) st.next(), buf.next();
            // A wait costs its latency even when nothing is left to wait for;
            // the next block's two are polled between its issue and its commits.
            // (With the two buffers of BN = 256 the next block's is this block's
            // own, which the commit below hands on: there that poll fails, and
            // the wait follows.)
            bool ready = false, free = first < Cfg::kBufs;
            int it = first;
            for (; it < total; it += 2) {
                if (!free && !wait(&acc_empty[buf.at], buf.parity ^ 1u)) break;
                if (!ready && !wait(&full[st.at], st.parity)) break;
                tc_fence_after();
                const uint32_t from = base + st.at * Cfg::kStageBytes;
                const uint64_t dp = sdesc_sw128(from, 16, 1024), dq = sdesc_sw128(from + kRows * kBk, 16, 1024);
#pragma unroll
                for (int ks = 0; ks < 4; ++ks)
                    mma_e4m3_pair(tmem + buf.at * BN, tc::desc_add(dp, 32 * ks), tc::desc_add(dq, 32 * ks), idesc,
                                  ks > 0);
                uint64_t *done = &acc_full[buf.at], *read = &empty[st.at];
                st.next(), st.next();
                buf.next(), buf.next();
                ready = it + 2 < total && mbar_try_wait(&full[st.at], st.parity);
                free = it + 2 < Cfg::kBufs || mbar_try_wait(&acc_empty[buf.at], buf.parity ^ 1u);
                mma_commit_pair(done);
                mma_commit_pair(read);
            }
            if (it < total) {
                mma_commit_pair(&drain[first]);
                mbar_wait(&drain[first], 0, tc::kWaitBudget);
            }
        } else if (QROWS && warp == 3) {
            // Scales: a row's of kPiece blocks lie side by side, and are read
            // together while their sectors are in L1 (one block at a time for
            // all rows, each would come from L2 again: L1 has what the stages
            // leave of it), in two pieces of 16 bytes where rows are aligned
            // to them (4096 x 4096 x 4096 by rows: 111 us, one by one 116).
            const int mine = pair < n_tiles ? (n_tiles - pair + pairs - 1) / pairs : 0;
            Ring<2> sc;
            int done = 0;
            bool ok = true;
            for (int i = 0; ok && i < mine; ++i) {
                int tp, tq;
                pair_tile(pair + i * pairs, tiles_p, a.tiles_q, &tp, &tq);
                for (int kb = 0; kb < nkb; kb += Cfg::kPiece, ++done) {
                    if (done >= 2 && !(ok = __all_sync(0xffffffffu, wait(&sc_empty[sc.at], sc.parity ^ 1u)))) break;
                    auto stage = [&](const Mm8Operand& o, int row, float* to, int pitch) {
                        const float* from = o.scale + (int64_t)(min(row, o.rows - 1) / o.per) * o.ld_scale + kb;
                        float v[Cfg::kPiece];
                        if (o.quads) {  // a piece of 4 is read if it holds a block that exists
                            const float4 lo = __ldg(reinterpret_cast<const float4*>(from));
                            const float4 up = __ldg(reinterpret_cast<const float4*>(from) + (kb + 4 < nkb));
                            v[0] = lo.x, v[1] = lo.y, v[2] = lo.z, v[3] = lo.w;
                            v[4] = up.x, v[5] = up.y, v[6] = up.z, v[7] = up.w;
                        } else {
#pragma unroll
                            for (int g = 0; g < Cfg::kPiece; ++g) v[g] = __ldg(from + min(g, nkb - 1 - kb));
                        }
#pragma unroll
                        for (int g = 0; g < Cfg::kPiece; ++g) to[g * pitch] = v[g];
                    };
#pragma unroll
                    for (int j = 0; j < kRows; j += 32)
                        stage(a.p, (2 * tp + rank) * kRows + j + lane, &row_scale[sc.at][0][j + lane], kRows);
#pragma unroll 4
                    for (int j = 0; j < BN; j += 32)
                        stage(a.q, tq * BN + j + lane, &col_scale[sc.at][0][j + lane], BN);
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sc_full[sc.at]);
                    sc.next();
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(QROWS ? 216 : 232));
        const int row = 32 * (warp & 3) + lane;      // of the tile
        const int c0 = (warp - 4) / 4 * Cfg::kRun;   // the warp's first column
        uint8_t* const staged = smem + Cfg::kStages * Cfg::kStageBytes + (warp - 4) * Cfg::kOuts * Cfg::kOutBytes;
        int turn = 0;                                // of the stagings
        const uint32_t lane_addr = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + (uint32_t)c0;
        bool alive = true;  // once a wait has run out no other is waited for, and the rest is garbage
        Ring<Cfg::kBufs> buf;
        Ring<2> sc;
        for (int tile = pair; tile < n_tiles; tile += pairs) {
            int tp, tq;
            pair_tile(tile, tiles_p, a.tiles_q, &tp, &tq);
            const int p0 = (2 * tp + rank) * kRows, q0 = tq * BN;
            // the scales of the row and of the columns that share one, two
            // blocks ahead (otherwise staged)
            const float* ps = a.p.scale + (int64_t)(min(p0 + row, a.p.rows - 1) / a.p.per) * a.p.ld_scale;
            const float* qs = a.q.scale + (int64_t)(min(q0 + c0, a.q.rows - 1) / a.q.per) * a.q.ld_scale;
            float ps_next = 0.0f, ps_then = 0.0f, qs_next = 0.0f, qs_then = 0.0f;
            if constexpr (!QROWS) {
                ps_next = __ldg(ps), ps_then = __ldg(ps + min(1, nkb - 1));
                qs_next = __ldg(qs), qs_then = __ldg(qs + min(1, nkb - 1));
            }
            uint64_t acc[Cfg::kRun / 2];
#pragma unroll
            for (int i = 0; i < Cfg::kRun / 2; ++i) acc[i] = 0;
            // 32 columns are read while the 32 before are added up
            uint32_t v[2][32];
            auto ld = [&](int c, uint32_t(&to)[32]) {
                if constexpr (QROWS)
                    tmem_ld_frag(lane_addr + buf.at * BN + c, to);
                else
                    tmem_ld(lane_addr + buf.at * BN + c, to);
            };
            bool loading = false;  // the block's first columns are on their way
            for (int kb = 0; kb < nkb; ++kb) {
                const int at = kb % Cfg::kPiece;
                uint64_t r2[QROWS ? 4 : 1];
                if constexpr (QROWS) {
                    if (at == 0 && alive) alive = __all_sync(0xffffffffu, wait(&sc_full[sc.at], sc.parity));
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float r = row_scale[sc.at][at][32 * (warp & 3) + 8 * j + lane / 4];
                        r2[j] = f2_of(r, r);
                    }
                } else {
                    const float r = ps_next * qs_next;
                    r2[0] = f2_of(r, r);
                    ps_next = ps_then;
                    ps_then = __ldg(ps + min(kb + 2, nkb - 1));
                    qs_next = qs_then;
                    qs_then = __ldg(qs + min(kb + 2, nkb - 1));
                }
                if (!loading) {
                    if (alive) alive = __all_sync(0xffffffffu, wait(&acc_full[buf.at], buf.parity));
                    tc_fence_after();
                    ld(0, v[0]);
                }
#pragma unroll
                for (int c = 0; c < Cfg::kRun; c += 32) {
                    uint32_t(&w)[32] = v[c / 32 & 1];
                    tmem_wait_ld(w);
                    if (c + 32 < Cfg::kRun) {
                        ld(c + 32, v[(c / 32 & 1) ^ 1]);
                    } else {  // all read
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive_cluster(cluster_addr(&acc_empty[buf.at], 0));
                        buf.next();
                        loading = QROWS && kb + 1 < nkb && __all_sync(0xffffffffu, mbar_test(&acc_full[buf.at], buf.parity));
                        if (loading) {
                            tc_fence_after();
                            ld(0, v[0]);
                        }
                    }
                    uint64_t cs[QROWS ? 4 : 1];
                    if constexpr (QROWS) {
#pragma unroll
                        for (int m = 0; m < 4; ++m) {
                            const float* at2 = &col_scale[sc.at][at][c0 + c + 8 * m + 2 * (lane & 3)];
                            const float2 f = *reinterpret_cast<const float2*>(at2);
                            cs[m] = f2_of(f.x, f.y);
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const uint64_t d = f2_of(__uint_as_float(w[2 * e]), __uint_as_float(w[2 * e + 1]));
                        uint64_t& o = acc[c / 2 + e];
                        if constexpr (QROWS)
                            o = f2_fma(d, f2_mul(r2[2 * (e / 8) + e % 2], cs[e / 2 % 4]), o);
                        else
                            o = f2_fma(d, r2[0], o);
                    }
                }
                if (QROWS && (at == Cfg::kPiece - 1 || kb == nkb - 1)) {
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sc_empty[sc.at]);
                    sc.next();
                }
            }
            // the warp's 32 rows: 128 bytes of each at a time through its
            // staging, then by TMA, or (out at any alignment) by the lanes
            constexpr int kPer = 128 / (int)sizeof(T);
            const int row0 = p0 + 32 * (warp & 3);
#pragma unroll
            for (int c = 0; c < Cfg::kRun; c += kPer) {
                // (lane 0) the last store from this staging has read it
                if constexpr (Cfg::kOuts == 2)
                    bulk_wait_read1();
                else
                    bulk_wait_read0();
                __syncwarp();
                const uint8_t* mine = staged + turn * Cfg::kOutBytes;
                const uint32_t staging = smem_u32(mine);
                turn = (turn + 1) % Cfg::kOuts;
                if constexpr (QROWS) {  // fragments
#pragma unroll
                    for (int e = 0; e < kPer / 2; ++e) {
                        const int r = 16 * (e / 8 % 2) + 8 * (e % 2) + lane / 4;
                        const int byte = (32 * (e / 16) + 8 * (e / 2 % 4) + 2 * (lane & 3)) * (int)sizeof(T);
                        const uint32_t to = staging + sw128_off(r, byte / 16) + byte % 16;
                        float lo, up;
                        f2_to(acc[c / 2 + e], lo, up);
                        if constexpr (sizeof(T) == 2)
                            asm volatile("st.shared.b32 [%0], %1;" ::"r"(to), "r"(bf16x2(lo, up)) : "memory");
                        else
                            asm volatile("st.shared.v2.f32 [%0], {%1, %2};" ::"r"(to), "f"(lo), "f"(up) : "memory");
                    }
                } else {
#pragma unroll
                    for (int u = 0; u < 8; ++u) {  // 16-byte units of the lane's row
                        uint32_t w[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            float lo, up;
                            if constexpr (sizeof(T) == 2) {
                                f2_to(acc[c / 2 + 4 * u + e], lo, up);
                                w[e] = bf16x2(lo, up);
                            } else {
                                f2_to(acc[c / 2 + 2 * u + e / 2], lo, up);
                                w[e] = __float_as_uint(e & 1 ? up : lo);
                            }
                        }
                        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(staging + sw128_off(lane, u)),
                                     "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3])
                                     : "memory");
                    }
                }
                const int col0 = q0 + c0 + c;
                if (a.vec_out) {
                    fence_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        if (row0 < a.p.rows && col0 < a.q.rows) tma_store_2d(&maps.out, staging, col0, row0);
                        bulk_commit();
                    }
                } else {
                    __syncwarp();
                    for (int r = 0; r < 32 && row0 + r < a.p.rows; ++r) {
                        T* o = static_cast<T*>(a.out) + (int64_t)(row0 + r) * a.ld_out + col0;
#pragma unroll
                        for (int e = lane; e < kPer; e += 32) {
                            const int at = e * (int)sizeof(T);
                            if (col0 + e < a.q.rows)
                                o[e] = *reinterpret_cast<const T*>(mine + sw128_off(r, at / 16) + at % 16);
                        }
                    }
                }
            }
        }
        bulk_wait0();
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();  // neither CTA leaves, or frees TMEM, under the other
    if (warp == 1) {
        tc_fence_after();
        tmem_free_pair(tmem, 512);
    }
}

struct Mm8Launch {
    cudaLaunchConfig_t  cfg{};
    cudaLaunchAttribute at{};
    Mm8Launch(int grid, int cluster, size_t smem, int threads, void* stream) {
        cfg.gridDim = dim3((unsigned)grid);
        cfg.blockDim = dim3((unsigned)threads);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = static_cast<cudaStream_t>(stream);
        at.id = cudaLaunchAttributeClusterDimension;
        at.val.clusterDim.x = (unsigned)cluster;
        at.val.clusterDim.y = at.val.clusterDim.z = 1;
        cfg.attrs = &at;
        cfg.numAttrs = 1;
    }
};

template <int BN, bool QROWS, typename T>
int launch_pair_t(const PairMaps& maps, const Mm8Params& p, int ctas, void* stream) {
    Mm8Launch l(ctas, 2, PairCfg<BN, QROWS>::kSmem, kPairThreads, stream);
    return cudaLaunchKernelEx(&l.cfg, mm8_pair_kernel<BN, QROWS, T>, maps, p);
}

template <int BN>
int launch_pair_n(bool qrows, helix_dtype out, const PairMaps& maps, const Mm8Params& p, int ctas, void* stream) {
    if (out == HELIX_F32)
        return qrows ? launch_pair_t<BN, true, float>(maps, p, ctas, stream)
                     : launch_pair_t<BN, false, float>(maps, p, ctas, stream);
    return qrows ? launch_pair_t<BN, true, __nv_bfloat16>(maps, p, ctas, stream)
                 : launch_pair_t<BN, false, __nv_bfloat16>(maps, p, ctas, stream);
}

template <int BN, bool QROWS>
int configure_pair_n() {
    const void* k[] = {(const void*)mm8_pair_kernel<BN, QROWS, float>,
                       (const void*)mm8_pair_kernel<BN, QROWS, __nv_bfloat16>};
    for (const void* f : k) {
        const int e =
            cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)PairCfg<BN, QROWS>::kSmem);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

template <int BN, bool QROWS, typename T>
int launch_mm8_t(const Mm8Maps& maps, const Mm8Params& p, int tiles, void* stream) {
    Mm8Launch l(tiles * p.splits, p.splits, Mm8Cfg<BN>::kSmem, kMmThreads, stream);
    return cudaLaunchKernelEx(&l.cfg, mm8_kernel<BN, QROWS, T>, maps, p);
}

template <int BN, bool QROWS>
int launch_mm8_n(helix_dtype out, const Mm8Maps& maps, const Mm8Params& p, int tiles, void* stream) {
    return out == HELIX_F32 ? launch_mm8_t<BN, QROWS, float>(maps, p, tiles, stream)
                            : launch_mm8_t<BN, QROWS, __nv_bfloat16>(maps, p, tiles, stream);
}

template <int BN, bool QROWS>
int configure_mm8_n() {
    const void* k[] = {(const void*)mm8_kernel<BN, QROWS, float>, (const void*)mm8_kernel<BN, QROWS, __nv_bfloat16>};
    for (const void* f : k) {
        const int e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Mm8Cfg<BN>::kSmem);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

// rows x k bytes in boxes of box_rows x 128, swizzled; zeros past the ends.
bool make_map_u8(const helix_ctx* ctx, CUtensorMap* m, const void* base, int64_t rows, int64_t k, int64_t ld,
                 int box_rows) {
    const auto fn = reinterpret_cast<tc::EncodeFn>(ctx->encode_tiled);
    if (rows == 1) ld = (k + 15) / 16 * 16;  // unused, but it has to be valid
    cuuint64_t dims[2] = {(cuuint64_t)k, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)ld};
    cuuint32_t box[2] = {(cuuint32_t)kBk, (cuuint32_t)box_rows};
    cuuint32_t es[2] = {1, 1};
    return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, es,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// out in boxes of 32 rows x 128 bytes, swizzled; what lies past the ends is not written.
bool make_map_out(const helix_ctx* ctx, CUtensorMap* m, void* base, int64_t rows, int64_t cols, int64_t ld,
                  helix_dtype type) {
    const auto fn = reinterpret_cast<tc::EncodeFn>(ctx->encode_tiled);
    const int size = type == HELIX_F32 ? 4 : 2;
    if (rows == 1) ld = (cols + 7) / 8 * 8;
    cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)(ld * size)};
    cuuint32_t box[2] = {(cuuint32_t)(128 / size), 32};
    cuuint32_t es[2] = {1, 1};
    return fn(m, size == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, base, dims, strides,
              box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int tiles_of(int64_t rows, int64_t per) { return (int)((rows + per - 1) / per); }

}  // namespace

int configure_mm8(helix_ctx* ctx) {
    int e;
    if ((e = configure_mm8_n<16, true>()) != cudaSuccess) return e;
    if ((e = configure_mm8_n<32, true>()) != cudaSuccess) return e;
    if ((e = configure_mm8_n<64, true>()) != cudaSuccess) return e;
    if ((e = configure_mm8_n<64, false>()) != cudaSuccess) return e;
    if ((e = configure_pair_n<128, true>()) != cudaSuccess) return e;
    if ((e = configure_pair_n<128, false>()) != cudaSuccess) return e;
    if ((e = configure_pair_n<256, true>()) != cudaSuccess) return e;
    if ((e = configure_pair_n<256, false>()) != cudaSuccess) return e;
    // clusters of 2, 4 and 8 that run at once with an SM for each CTA
    static_assert(Mm8Cfg<64>::kPerSm == 1, "");
    for (int i = 0; i < 3; ++i) {
        Mm8Launch l(2 << i, 2 << i, Mm8Cfg<64>::kSmem, kMmThreads, nullptr);
        e = cudaOccupancyMaxActiveClusters(&ctx->mm8_clusters[i], mm8_kernel<64, true, float>, &l.cfg);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

// Few rows of a become the MMA's columns (swap).  Where whole tiles leave SMs
// idle, a tile's blocks of k go to a cluster of CTAs, at least 4 blocks each
// (64 x 4096 x 1024: 8.0 us with 8 blocks each, 7.5 with 4, 8.2 with 2; 16 x
// 1024 x 4096: 8.2 with 16, 6.9 with 8, 6.7 with 4), while each CTA still has an
// SM of its own (16 x 8192 x 4096: 11.0 us with 64 CTAs, 8.3 with 128, 13.2 with
// 256; 16 x 2048 x 8192: 8.9 in clusters of 4, 14.0 in 16 clusters of 8, which
// the GPCs do not hold at once).  Products with more tiles than SMs run on pairs
// of CTAs, on the tile with the shorter estimate: waves of pairs times the
// measured time of a block of k, plus the start and end of a tile (128 wide
// where 256 leaves pairs idle, 512 x 4096 x 4096: 15.5 us against 21.1; else 256,
// 8192 x 8192 x 4096: 258 against 304).
Mm8Plan mm8_plan(const helix_ctx* ctx, const helix_matmul8_desc& d) {
    Mm8Plan pl{};
    pl.swap = d.m <= 64;
    pl.bn = !pl.swap ? 64 : d.m <= 16 ? 16 : d.m <= 32 ? 32 : 64;
    const int64_t tiles = (int64_t)tiles_of(pl.swap ? d.n : d.m, kRows) * tiles_of(pl.swap ? d.m : d.n, pl.bn);
    const int kb = tiles_of(d.k, kBk);
    pl.splits = 1;
    for (int i = 0; i < 3 && tiles <= ctx->mm8_clusters[i] && kb >= 4 << (i + 1); ++i) pl.splits = 2 << i;
    if (pl.swap || tiles <= ctx->n_sm) return pl;
    const bool rows = d.b_form == HELIX_SCALE_ROWS;
    auto estimate = [&](int bn, double block, double tile) {
        const int64_t n = (int64_t)tiles_of(d.m, 2 * kRows) * tiles_of(d.n, bn);
        const int64_t waves = (n + ctx->n_sm / 2 - 1) / (ctx->n_sm / 2);
        return (double)waves * (block * kb + tile);  // us
    };
    const double wide = rows ? estimate(256, 0.65, 4.3) : estimate(256, 0.49, 2.6);
    const double narrow = rows ? estimate(128, 0.45, 2.0) : estimate(128, 0.29, 1.7);
    pl.pair = true;
    pl.bn = wide <= narrow ? 256 : 128;
    return pl;
}

int launch_mm8(const helix_ctx* ctx, const helix_matmul8_desc& d, const Mm8Plan& pl, Mm8Params p, const void* a,
               const void* b, void* stream) {
    if (pl.pair) {
        PairMaps maps;
        std::memset(&maps, 0, sizeof(maps));
        if (!make_map_u8(ctx, &maps.p, a, d.m, d.k, d.ld_a, kRows) ||
            !make_map_u8(ctx, &maps.q, b, d.n, d.k, d.ld_b, pl.bn / 2) ||
            (p.vec_out && !make_map_out(ctx, &maps.out, p.out, d.m, d.n, d.ld_out, d.out_dtype)))
            return cudaErrorInvalidValue;
        p.tiles_q = tiles_of(d.n, pl.bn);
        const int64_t tiles = (int64_t)tiles_of(d.m, 2 * kRows) * p.tiles_q;
        // a pair counts its blocks of k in 32 bits
        if (tiles > INT32_MAX / 2 || (tiles / (ctx->n_sm / 2) + 1) * p.k_blocks > INT32_MAX)
            return cudaErrorInvalidValue;
        const int ctas = 2 * (int)std::min<int64_t>(tiles, ctx->n_sm / 2);
        return pl.bn == 256 ? launch_pair_n<256>(p.q.per == 1, d.out_dtype, maps, p, ctas, stream)
                            : launch_pair_n<128>(p.q.per == 1, d.out_dtype, maps, p, ctas, stream);
    }
    Mm8Maps maps;
    std::memset(&maps, 0, sizeof(maps));
    const bool ok = pl.swap ? make_map_u8(ctx, &maps.p, b, d.n, d.k, d.ld_b, kRows) &&
                                  make_map_u8(ctx, &maps.q, a, d.m, d.k, d.ld_a, pl.bn)
                            : make_map_u8(ctx, &maps.p, a, d.m, d.k, d.ld_a, kRows) &&
                                  make_map_u8(ctx, &maps.q, b, d.n, d.k, d.ld_b, pl.bn);
    if (!ok) return cudaErrorInvalidValue;
    p.tiles_q = tiles_of(p.q.rows, pl.bn);
    const int64_t tiles = (int64_t)tiles_of(p.p.rows, kRows) * p.tiles_q;
    if (tiles * p.splits > INT32_MAX) return cudaErrorInvalidValue;
    // narrow tiles have rows of a for columns, each with its own scales
    if (pl.bn == 16) return launch_mm8_n<16, true>(d.out_dtype, maps, p, (int)tiles, stream);
    if (pl.bn == 32) return launch_mm8_n<32, true>(d.out_dtype, maps, p, (int)tiles, stream);
    return p.q.per == 1 ? launch_mm8_n<64, true>(d.out_dtype, maps, p, (int)tiles, stream)
                        : launch_mm8_n<64, false>(d.out_dtype, maps, p, (int)tiles, stream);
}

}  // namespace hx
