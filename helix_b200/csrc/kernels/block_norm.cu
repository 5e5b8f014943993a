// block_norm.cu -- root-mean-square norm with the residual's addition, its
// output in 8 bits or not, and its gradient.
//
//     s = x + r,  rstd = 1 / sqrt(mean(s^2) + eps),  n = s rstd w
//     ds = dsum + rstd (dn w - s rstd^2 mean(dn w s)),  dw = sum_rows dn s rstd
//
// Both are bound by memory: one pass, the row kept in registers between its
// statistic and its output.  A row belongs to wpr warps; a warp holds V
// segments of 256 columns (segment j * wpr + warp), a lane 8 values of each.
// With vector accesses a lane's 8 values are consecutive, so 16 lanes hold a
// group of 128; without (odd widths or strides) lane l holds columns l + 32 e
// of the segment, so every access is still a run of 32 values, and the whole
// warp holds each of the segment's two groups.
//
// Sums, statistics and the products are fp32 (the row's mean by a rounded
// 1 / n_col, rstd by rsqrtf); to fewer bits go the stored sum and the output
// alone.  In 8 bits a value is multiplied by an approximate 1 / scale.
//
// What bounds them beside memory is the instructions: three quarters of the
// issue slots before the arithmetic went in pairs (fp32 x 2) and the
// gradient's rows came by asynchronous copies, its weights in registers.
//
// Measured: 8192 x 4096 bf16 to bf16 43.5 us, 6.2 TB/s, to 8 bits, where a
// group's maximum and scale come between the row's statistic and its output,
// 44.4, 5.3; f32 82, 6.5; 1537 x 2501 f32 10.9,
// 5.6; 8192 x 8192 bf16 87, 4096 x 16384 87; gradient of 16384 x 4096 bf16 88.5
// us, 6.1 TB/s (a copy's rate is 6.55), of 8192 x 4096 f32 96, 5.6; of 8192 x
// 4095, whose rows start anywhere, bf16 78, f32 98.
#include <algorithm>

#include "block_common.cuh"
#include "umma.cuh"

namespace hx {
namespace {

using umma::f2_add, umma::f2_fma, umma::f2_mul, umma::f2_of, umma::f2_of_bf16x2, umma::f2_to;

constexpr int kSeg = 256;        // columns of a warp's segment
constexpr int kMaxWarps = 32;    // 32 warps x 2 segments x 256 = 16384 columns

template <bool VEC>
__device__ __forceinline__ int col_of(int c0, int lane, int e) {
    return VEC ? c0 + 8 * lane + e : c0 + 32 * e + lane;
}

// The lane's 8 values of the segment at c0, 0 past the row's end; loaded
// first and looked at later.
template <bool VEC, typename T>
struct Seg {
    Raw8<T> raw;
    T       one[VEC ? 1 : 8];
    __device__ __forceinline__ void load(const T* row, int c0, int lane, int n_col) {
        if constexpr (VEC) {
            raw.zero();
            if (c0 + 8 * lane + 8 <= n_col) raw.load(row + c0 + 8 * lane);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int c = col_of<VEC>(c0, lane, e);
                one[e] = c < n_col ? row[c] : from_f32<T>(0.0f);
            }
        }
    }
    // as pairs of consecutive e
    __device__ __forceinline__ void get(const T* row, int c0, int lane, int n_col, uint64_t (&v)[4]) const {
        if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (sizeof(T) == 2) {
                    const uint32_t w[4] = {raw.v[0].x, raw.v[0].y, raw.v[0].z, raw.v[0].w};
                    v[i] = f2_of_bf16x2(w[i]);
                } else {
                    const uint4 q = raw.v[i / 2];
                    v[i] = i % 2 ? f2_of(__uint_as_float(q.z), __uint_as_float(q.w))
                                 : f2_of(__uint_as_float(q.x), __uint_as_float(q.y));
                }
            }
            // a row's last values where they are no whole eight
            const int c = c0 + 8 * lane;
            if (c < n_col && c + 8 > n_col) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    v[i] = f2_of(c + 2 * i < n_col ? to_f32(row[c + 2 * i]) : 0.0f,
                                 c + 2 * i + 1 < n_col ? to_f32(row[c + 2 * i + 1]) : 0.0f);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = f2_of(to_f32(one[2 * i]), to_f32(one[2 * i + 1]));
        }
    }
};
__device__ __forceinline__ void to_8(const uint64_t (&p)[4], float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f2_to(p[i], v[2 * i], v[2 * i + 1]);
}
template <bool VEC, typename T>
__device__ __forceinline__ void st_seg(T* row, int c0, int lane, int n_col, const uint64_t (&p)[4]) {
    float v[8];
    to_8(p, v);
    if (VEC && c0 + 8 * lane + 8 <= n_col) {
        st8(row + c0 + 8 * lane, v);
        return;
    }
    if (!VEC && c0 + kSeg <= n_col) {
#pragma unroll
        for (int e = 0; e < 8; ++e) row[c0 + 32 * e + lane] = from_f32<T>(v[e]);
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int c = col_of<VEC>(c0, lane, e);
        if (c < n_col) row[c] = from_f32<T>(v[e]);
    }
}
template <bool VEC, typename T>
__device__ __forceinline__ void ld_seg(const T* row, int c0, int lane, int n_col, uint64_t (&v)[4]) {
    Seg<VEC, T> s;
    s.load(row, c0, lane, n_col);
    s.get(row, c0, lane, n_col, v);
}
template <bool VEC>
__device__ __forceinline__ void ld_weight(const NormParams& p, int c0, int lane, uint64_t (&v)[4]) {
    if (p.w_bf16)
        ld_seg<VEC>(static_cast<const __nv_bfloat16*>(p.w), c0, lane, p.n_col, v);
    else
        ld_seg<VEC>(static_cast<const float*>(p.w), c0, lane, p.n_col, v);
}

// Starts the segment at c0 on its way to L2.
template <typename T>
__device__ __forceinline__ void prefetch_seg(const T* row, int c0, int lane, int n_col) {
    constexpr int kLanes = 128 / 8 / (int)sizeof(T);  // lanes whose 8 values make a line
    const int c = c0 + 8 * lane;
    if (lane % kLanes == 0 && c < n_col) asm volatile("prefetch.global.L2 [%0];" ::"l"(row + c));
}

__device__ __forceinline__ float both(uint64_t v) {
    float a, b;
    f2_to(v, a, b);
    return a + b;
}

// Sum over the wpr warps of a row (every warp of the block calls it).
// `part` holds one float per warp; buffers alternate between calls so that
// one barrier a call is enough.
__device__ __forceinline__ float row_sum(float v, int wpr, int warp, int lane, float* part) {
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (wpr == 1) return v;
    if (lane == 0) part[warp] = v;
    __syncthreads();
    v = lane < wpr ? part[warp / wpr * wpr + lane] : 0.0f;
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// The segment's 8 values a lane holds, as e4m3 with its group's scale.
template <bool VEC>
__device__ __forceinline__ void st_seg_e4m3(const NormParams& p, int64_t row, int c0, int lane,
                                            const uint64_t (&pairs)[4]) {
    uint8_t* q = static_cast<uint8_t*>(p.out) + row * p.ld_out;
    float* sc = p.scale + row * p.ld_scale;
    float n[8];
    to_8(pairs, n);
    if constexpr (VEC) {
        float a = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) a = max_abs_nan(a, n[2 * i], n[2 * i + 1]);
#pragma unroll
        for (int o = 8; o >= 1; o >>= 1) a = max_nan(a, __shfl_xor_sync(0xffffffffu, a, o));
        float inv;
        const float scale = group_scale(a, &inv);
        const int c = c0 + 8 * lane;
        if ((lane & 15) == 0 && c < p.n_col) sc[c / HELIX_GROUP] = scale;
        const uint64_t inv2 = f2_of(inv, inv);
        uint64_t r[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = f2_mul(pairs[i], inv2);
        to_8(r, n);
        if (c + 8 <= p.n_col) {
            *reinterpret_cast<uint2*>(q + c) = make_uint2(e4m3x2(n[0], n[1]) | e4m3x2(n[2], n[3]) << 16,
                                                          e4m3x2(n[4], n[5]) | e4m3x2(n[6], n[7]) << 16);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (c + e < p.n_col) q[c + e] = (uint8_t)e4m3x2(n[e], 0.0f);
        }
    } else {
#pragma unroll
        for (int g = 0; g < 2; ++g) {  // the segment's groups: e = 0..3 and 4..7
            float a = 0.0f;
#pragma unroll
            for (int e = 4 * g; e < 4 * g + 4; e += 2) a = max_abs_nan(a, n[e], n[e + 1]);
#pragma unroll
            for (int o = 16; o >= 1; o >>= 1) a = max_nan(a, __shfl_xor_sync(0xffffffffu, a, o));
            float inv;
            const float scale = group_scale(a, &inv);
            const int first = c0 + HELIX_GROUP * g;
            if (lane == 0 && first < p.n_col) sc[first / HELIX_GROUP] = scale;
#pragma unroll
            for (int e = 4 * g; e < 4 * g + 4; ++e) {
                const int c = c0 + 32 * e + lane;
                if (c < p.n_col) q[c] = (uint8_t)e4m3x2(n[e] * inv, 0.0f);
            }
        }
    }
}

// One row.  `part` holds one float per warp.
template <typename TX, typename TR, int V, bool VEC>
__device__ __forceinline__ void norm_row(const NormParams& p, int64_t row, bool live, int warp, int lane, float* part) {
    const int wr = warp % p.wpr;
    const int n = live ? p.n_col : 0;
    const TX* x = static_cast<const TX*>(p.x) + (live ? row : 0) * p.ld_x;
    const TR* r = static_cast<const TR*>(p.res) + (live ? row : 0) * p.ld_res;

    uint64_t s[V][4], ss2 = 0;
    {
        Seg<VEC, TX> sx[V];
        Seg<VEC, TR> sr[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int c0 = (j * p.wpr + wr) * kSeg;
            sx[j].load(x, c0, lane, n);
            sr[j].load(r, c0, lane, p.res ? n : 0);
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int c0 = (j * p.wpr + wr) * kSeg;
            uint64_t v[4];
            sx[j].get(x, c0, lane, n, s[j]);
            sr[j].get(r, c0, lane, p.res ? n : 0, v);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (p.res) s[j][i] = f2_add(s[j][i], v[i]);
                ss2 = f2_fma(s[j][i], s[j][i], ss2);
            }
        }
    }
    const float ss = row_sum(both(ss2), p.wpr, warp, lane, part);
    if (!live) return;
    const float rstd = rsqrtf(ss * p.inv_col + p.eps);
    if (p.rstd && wr == 0 && lane == 0) p.rstd[row] = rstd;
    const uint64_t rstd2 = f2_of(rstd, rstd);

#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int c0 = (j * p.wpr + wr) * kSeg;
        if (p.sum) st_seg<VEC>(static_cast<TR*>(p.sum) + row * p.ld_sum, c0, lane, p.n_col, s[j]);
        uint64_t w[4];
        ld_weight<VEC>(p, c0, lane, w);
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = f2_mul(w[i], f2_mul(s[j][i], rstd2));
        if (p.out_dtype == HELIX_E4M3)
            st_seg_e4m3<VEC>(p, row, c0, lane, w);
        else if (p.out_dtype == HELIX_BF16)
            st_seg<VEC>(static_cast<__nv_bfloat16*>(p.out) + row * p.ld_out, c0, lane, p.n_col, w);
        else
            st_seg<VEC>(static_cast<float*>(p.out) + row * p.ld_out, c0, lane, p.n_col, w);
    }
}

// 48 registers, so that five blocks fit an SM (8192 x 4096 bf16 to 8 bits: 44.4
// us, with four 48.4; six spill, 8192 x 4096 f32: 82 -> 102).
template <typename TX, typename TR, int V, bool VEC>
__global__ void __launch_bounds__(256, 5) norm_kernel(const NormParams p) {
    __shared__ float part[8];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t row = (int64_t)blockIdx.x * p.rpb + warp / p.wpr;
    norm_row<TX, TR, V, VEC>(p, row, row < p.n_row, warp, lane, part);
}

// Rows of more than 8 warps: too few blocks fit an SM for one's loads to
// cover another's barrier, so blocks stay and send their next row to L2 first.
template <typename TX, typename TR, bool VEC>
__global__ void __launch_bounds__(1024, 1) norm_wide_kernel(const NormParams p) {
    __shared__ float part[2][kMaxWarps];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int turn = 0;
    for (int64_t row = blockIdx.x; row < p.n_row; row += gridDim.x) {
        const int64_t next = row + gridDim.x;
        if (next < p.n_row) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int c0 = (j * p.wpr + warp) * kSeg;
                prefetch_seg(static_cast<const TX*>(p.x) + next * p.ld_x, c0, lane, p.n_col);
                if (p.res) prefetch_seg(static_cast<const TR*>(p.res) + next * p.ld_res, c0, lane, p.n_col);
            }
        }
        norm_row<TX, TR, 2, VEC>(p, row, true, warp, lane, part[turn]);
        turn ^= 1;
    }
}

// Asynchronous copy of 16 bytes to shared memory, or zeros.
__device__ __forceinline__ void copy16(uint32_t to, const void* from, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Rows on their way to a gradient's warps, kGradStages of them: a tensor's segment
// of 256 columns in shared memory of the warp's own, which nobody else reads,
// so no barrier.  Lanes copy consecutive 16-byte pieces: of the segment's whole
// pieces with vector accesses (with 2-byte types those that a lane reads back
// itself), else all that hold a part of the segment at whatever offset, each of
// which holds a value that exists.  They keep their place in a line of 128
// bytes, so that a warp's 512 are 4 lines (8192 x 4095 f32: 98 us, as 5 lines 110).
template <typename T, bool VEC>
struct Ahead {
    static constexpr int kLine = 128, kBytes = kSeg * (int)sizeof(T) + (VEC ? 0 : kLine);
    static __device__ __forceinline__ void copy(uint32_t to, const T* row, int c0, int lane, int n_col) {
        if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < kBytes; i += 512) {
                const int  c = c0 + (i + 16 * lane) / (int)sizeof(T);
                const bool live = c + 16 / (int)sizeof(T) <= n_col;
                copy16(to + i + 16 * lane, row + (live ? c : 0), live);
            }
        } else {
            const uintptr_t at = reinterpret_cast<uintptr_t>(row + c0);
            const int bytes = min(n_col - c0, kSeg) * (int)sizeof(T), off = (int)(at & (kLine - 1));
#pragma unroll
            for (int i = 0; i < kBytes; i += 512) {
                const int b = i + 16 * lane;
                if (b > off - 16 && b < off + bytes)
                    copy16(to + b, reinterpret_cast<const void*>(at - off + b), true);
            }
        }
    }
    static __device__ __forceinline__ void take(const uint8_t* from, const T* row, int c0, int lane, int n_col,
                                                Seg<VEC, T>& s) {
        if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; ++i)
                s.raw.v[i] = *reinterpret_cast<const uint4*>(from + 8 * (int)sizeof(T) * lane + 16 * i);
        } else {
            const T* at = reinterpret_cast<const T*>(from + (reinterpret_cast<uintptr_t>(row + c0) & (kLine - 1)));
            if (c0 + kSeg <= n_col) {
#pragma unroll
                for (int e = 0; e < 8; ++e) s.one[e] = at[32 * e + lane];
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    s.one[e] = c0 + 32 * e + lane < n_col ? at[32 * e + lane] : from_f32<T>(0.0f);
            }
        }
    }
};
constexpr int kGradStages = 2;  // (turn alternates)
// Of a warp, for dout, sum and dsum.
template <typename TX, typename TR, bool VEC>
constexpr int kAheadBytes = Ahead<TX, VEC>::kBytes + 2 * Ahead<TR, VEC>::kBytes;

// Persistent: a row slot takes every slots-th row and keeps its share of
// dweight in registers, written to partial[slot] at the end.
template <typename TX, typename TR, int V, bool VEC>
__global__ void __launch_bounds__(V == 1 ? 1024 : 512, 1) norm_grad_kernel(const NormParams p) {
    __shared__ float part[2][kMaxWarps];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rg = warp / p.wpr, wr = warp % p.wpr;
    // The widest rows (V = 4) leave no registers for dweight, which then stays
    // in shared memory, nor for the weights, and no room for rows ahead.
    constexpr bool kWide = V == 4;
    // lanes read what others copied
    constexpr bool kShared = !VEC || sizeof(TX) == 4 || sizeof(TR) == 4;
    // 4-byte values, or single accesses, leave no registers for dsum's before it is used
    constexpr bool kLate = kShared;
    extern __shared__ __align__(16) uint8_t smem[];
    uint64_t dw[kWide ? 1 : V][4];
    auto dw_at = [&](int j, int i) -> uint64_t& {
        if constexpr (kWide)
            return reinterpret_cast<uint64_t*>(smem)[(4 * j + i) * blockDim.x + threadIdx.x];
        else
            return dw[j][i];
    };
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) dw_at(j, i) = 0;

    const TX* dout = static_cast<const TX*>(p.dout);
    const TR* sum = static_cast<const TR*>(p.sum);
    const TR* dsum = static_cast<const TR*>(p.dsum);
    Seg<VEC, TX> sd[V];
    Seg<VEC, TR> ss[V];
    uint64_t weight[4];
    float    rstd_next = 0.0f;
    const int64_t step = (int64_t)gridDim.x * p.rpb;

    // rows ahead (not kWide)
    uint8_t* const ahead = smem + warp * kGradStages * kAheadBytes<TX, TR, VEC>;
    auto copy = [&](int64_t row, int stage) {
        const int n = row < p.n_row ? p.n_col : 0, c0 = wr * kSeg;
        row = n ? row : 0;
        const uint32_t to = (uint32_t)__cvta_generic_to_shared(ahead + stage * kAheadBytes<TX, TR, VEC>);
        Ahead<TX, VEC>::copy(to, dout + row * p.ld_dout, c0, lane, n);
        Ahead<TR, VEC>::copy(to + Ahead<TX, VEC>::kBytes, sum + row * p.ld_sum, c0, lane, n);
        if (dsum)
            Ahead<TR, VEC>::copy(to + Ahead<TX, VEC>::kBytes + Ahead<TR, VEC>::kBytes, dsum + row * p.ld_dsum, c0, lane,
                                 n);
        copies_commit();
    };
    auto take = [&](int64_t row, int stage, int n) {
        const int c0 = wr * kSeg;
        const uint8_t* from = ahead + stage * kAheadBytes<TX, TR, VEC>;
        if (kShared) __syncwarp();
        Ahead<TX, VEC>::take(from, dout + row * p.ld_dout, c0, lane, n, sd[0]);
        Ahead<TR, VEC>::take(from + Ahead<TX, VEC>::kBytes, sum + row * p.ld_sum, c0, lane, n, ss[0]);
    };
    auto take_dsum = [&](int64_t row, int stage, int n, uint64_t (&v)[4]) {
        const int c0 = wr * kSeg;
        const uint8_t* from = ahead + stage * kAheadBytes<TX, TR, VEC>;
        Seg<VEC, TR> sa;
        if (dsum)
            Ahead<TR, VEC>::take(from + Ahead<TX, VEC>::kBytes + Ahead<TR, VEC>::kBytes, dsum + row * p.ld_dsum, c0,
                                 lane, n, sa);
        else
            sa.load(dsum, c0, lane, 0);  // zeros
        sa.get(dsum + row * p.ld_dsum, c0, lane, dsum ? n : 0, v);
    };
    if constexpr (!kWide) {
        ld_weight<VEC>(p, wr * kSeg, lane, weight);
        const int64_t first = (int64_t)blockIdx.x * p.rpb + rg;
        for (int k = 0; k < kGradStages; ++k) copy(first + k * step, k);
        rstd_next = first < p.n_row ? p.rstd[first] : 0.0f;
    }

    int turn = 0;
    for (int64_t base = (int64_t)blockIdx.x * p.rpb; base < p.n_row; base += step) {
        const bool live = base + rg < p.n_row;
        const int64_t row = live ? base + rg : 0;
        const int n = live ? p.n_col : 0;
        float rstd = rstd_next;
        uint64_t o[4];
        if constexpr (kWide) {
            rstd = live ? p.rstd[row] : 0.0f;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const int c0 = (j * p.wpr + wr) * kSeg;
                sd[j].load(dout + row * p.ld_dout, c0, lane, n);
                ss[j].load(sum + row * p.ld_sum, c0, lane, n);
            }
            if (base + step < p.n_row) {  // the next row goes to L2
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const int c0 = (j * p.wpr + wr) * kSeg;
                    prefetch_seg(dout + (base + step) * p.ld_dout, c0, lane, p.n_col);
                    prefetch_seg(sum + (base + step) * p.ld_sum, c0, lane, p.n_col);
                    if (p.dsum) prefetch_seg(dsum + (base + step) * p.ld_dsum, c0, lane, p.n_col);
                }
            }
        } else {
            const int64_t next = base + step + rg;
            copies_wait<kGradStages - 1>();
            take(row, turn, n);
            rstd_next = next < p.n_row ? p.rstd[next] : 0.0f;
            if constexpr (!kLate) {
                take_dsum(row, turn, n, o);
                copy(next + (kGradStages - 1) * step, turn);
            }
        }
        const uint64_t rstd2 = f2_of(rstd, rstd);
        uint64_t d[V][4], s[V][4], along2 = 0;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int c0 = (j * p.wpr + wr) * kSeg;
            sd[j].get(dout + row * p.ld_dout, c0, lane, n, d[j]);
            ss[j].get(sum + row * p.ld_sum, c0, lane, n, s[j]);
            if constexpr (kWide) ld_weight<VEC>(p, c0, lane, weight);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[j][i] = f2_mul(s[j][i], rstd2);      // s rstd
                dw_at(j, i) = f2_fma(d[j][i], s[j][i], dw_at(j, i));
                d[j][i] = f2_mul(d[j][i], weight[i]);  // dn w
                along2 = f2_fma(d[j][i], s[j][i], along2);
            }
        }
        const float along = -row_sum(both(along2), p.wpr, warp, lane, part[turn]) * p.inv_col;
        along2 = f2_of(along, along);
        if constexpr (!kWide && kLate) {
            take_dsum(row, turn, n, o);
            __syncwarp();
            copy(base + kGradStages * step + rg, turn);
        }
        turn ^= 1;
        if (!live) continue;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int c0 = (j * p.wpr + wr) * kSeg;
            if constexpr (kWide) ld_seg<VEC>(dsum + row * p.ld_dsum, c0, lane, p.dsum ? n : 0, o);
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = f2_fma(rstd2, f2_fma(s[j][i], along2, d[j][i]), o[i]);
            st_seg<VEC>(static_cast<TX*>(p.dx) + row * p.ld_dx, c0, lane, n, o);
            if (p.dres) st_seg<VEC>(static_cast<TR*>(p.dres) + row * p.ld_dres, c0, lane, n, o);
        }
    }
    umma::grid_dep_launch();
    float* mine = p.partial + ((int64_t)blockIdx.x * p.rpb + rg) * p.n_col;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int c0 = (j * p.wpr + wr) * kSeg;
        float v[8];
        const uint64_t pairs[4] = {dw_at(j, 0), dw_at(j, 1), dw_at(j, 2), dw_at(j, 3)};
        to_8(pairs, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int c = col_of<VEC>(c0, lane, e);
            if (c < p.n_col) mine[c] = v[e];
        }
    }
}

// dweight[c] = the partials' sum in the order of the slots.  Its blocks may
// start as the gradient's end (a programmatic dependent launch), and wait for
// all of them.
constexpr int kDwRows = 32;
__global__ void __launch_bounds__(32 * kDwRows) norm_dw_kernel(const float* partial, int slots, int n_col,
                                                              float* dweight) {
    __shared__ float part[kDwRows][33];
    const int lane = threadIdx.x & 31, r = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + lane;
    umma::grid_dep_wait();
    float v = 0.0f;
    if (c < n_col)
#pragma unroll 10
        for (int s = r; s < slots; s += kDwRows) v += partial[(int64_t)s * n_col + c];
    part[r][lane] = v;
    __syncthreads();
    if (r == 0 && c < n_col) {
#pragma unroll
        for (int i = 1; i < kDwRows; ++i) v += part[i][lane];
        dweight[c] = v;
    }
}

constexpr size_t kWideSmem = sizeof(float) * 32 * 512;  // dweight of a block's row at V = 4

template <typename TX, typename TR, bool VEC>
int launch_norm_v(const NormParams& p, int v, dim3 grid, dim3 block, bool grad, void* stream) {
    if (grad)
        return v == 1 ? block_launch(norm_grad_kernel<TX, TR, 1, VEC>, grid, block,
                                     block.x / 32 * kGradStages * kAheadBytes<TX, TR, VEC>, stream, p)
                      : block_launch(norm_grad_kernel<TX, TR, 4, VEC>, grid, block, kWideSmem, stream, p);
    if (block.x > 256) return block_launch(norm_wide_kernel<TX, TR, VEC>, grid, block, 0, stream, p);
    return v == 1 ? block_launch(norm_kernel<TX, TR, 1, VEC>, grid, block, 0, stream, p)
                  : block_launch(norm_kernel<TX, TR, 2, VEC>, grid, block, 0, stream, p);
}

int launch_norm_any(const helix_rms_norm_desc& d, const NormParams& p, int v, dim3 grid, dim3 block, bool vec,
                    bool grad, void* stream) {
    using bf = __nv_bfloat16;
    if (d.x_dtype == HELIX_F32)
        return vec ? launch_norm_v<float, float, true>(p, v, grid, block, grad, stream)
                   : launch_norm_v<float, float, false>(p, v, grid, block, grad, stream);
    if (d.sum_dtype == HELIX_F32)
        return vec ? launch_norm_v<bf, float, true>(p, v, grid, block, grad, stream)
                   : launch_norm_v<bf, float, false>(p, v, grid, block, grad, stream);
    return vec ? launch_norm_v<bf, bf, true>(p, v, grid, block, grad, stream)
               : launch_norm_v<bf, bf, false>(p, v, grid, block, grad, stream);
}

template <typename TX, typename TR, bool VEC>
int configure_norm_t() {
    const int e = cudaFuncSetAttribute(norm_grad_kernel<TX, TR, 1, VEC>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       kMaxWarps * kGradStages * kAheadBytes<TX, TR, VEC>);
    if (e != cudaSuccess) return e;
    return cudaFuncSetAttribute(norm_grad_kernel<TX, TR, 4, VEC>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                (int)kWideSmem);
}

}  // namespace

int configure_norm() {
    using bf = __nv_bfloat16;
    int e;
    if ((e = configure_norm_t<float, float, true>()) != cudaSuccess) return e;
    if ((e = configure_norm_t<float, float, false>()) != cudaSuccess) return e;
    if ((e = configure_norm_t<bf, float, true>()) != cudaSuccess) return e;
    if ((e = configure_norm_t<bf, float, false>()) != cudaSuccess) return e;
    if ((e = configure_norm_t<bf, bf, true>()) != cudaSuccess) return e;
    return configure_norm_t<bf, bf, false>();
}

namespace {

NormShape shape_of(int n_col, int v) {
    NormShape s{};
    s.v = v;
    s.wpr = ((n_col + kSeg - 1) / kSeg + v - 1) / v;
    s.rpb = s.wpr >= 8 ? 1 : 8 / s.wpr;
    return s;
}

}  // namespace

NormShape norm_shape(const helix_rms_norm_desc& d) { return shape_of(d.n_col, d.n_col <= kSeg ? 1 : 2); }

// The gradient has one segment per warp, the most rows in flight that 64
// registers allow; the widest rows have four (32 warps cover no more with one).
NormGradPlan norm_grad_plan(const helix_ctx* ctx, const helix_rms_norm_desc& d) {
    NormGradPlan pl{};
    const int segs = (d.n_col + kSeg - 1) / kSeg;
    pl.shape = shape_of(d.n_col, segs > 32 ? 4 : 1);
    const int n_sm = ctx && ctx->n_sm > 0 ? ctx->n_sm : 148;
    // blocks that the registers of an SM allow
    const int64_t per_sm = std::max((pl.shape.v == 1 ? 32 : 16) / (pl.shape.wpr * pl.shape.rpb), 1);
    const int64_t need = (d.n_row + pl.shape.rpb - 1) / pl.shape.rpb;
    pl.blocks = (int)std::min(need, n_sm * per_sm);
    pl.slots = pl.blocks * pl.shape.rpb;
    pl.total = ((size_t)pl.slots * (size_t)d.n_col * sizeof(float) + 255) & ~(size_t)255;
    return pl;
}

int launch_norm(const helix_ctx* ctx, const helix_rms_norm_desc& d, const NormParams& p, bool vec, void* stream) {
    const NormShape s = norm_shape(d);
    const dim3 block(32 * s.wpr * s.rpb);
    int64_t blocks = (d.n_row + s.rpb - 1) / s.rpb;
    if (block.x > 256) blocks = std::min<int64_t>(blocks, (int64_t)ctx->n_sm * (block.x > 512 ? 1 : 2));
    const dim3 grid((unsigned)blocks);
    return launch_norm_any(d, p, s.v, grid, block, vec, false, stream);
}

int launch_norm_grad(const helix_rms_norm_desc& d, const NormGradPlan& pl, const NormParams& p, bool vec,
                     float* dweight, void* stream) {
    if (pl.blocks > 0) {
        const dim3 grid((unsigned)pl.blocks), block(32 * pl.shape.wpr * pl.shape.rpb);
        const int e = launch_norm_any(d, p, pl.shape.v, grid, block, vec, true, stream);
        if (e != cudaSuccess) return e;
    }
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute early{};
    cfg.gridDim = dim3((unsigned)((d.n_col + 31) / 32));
    cfg.blockDim = dim3(32 * kDwRows);
    cfg.stream = static_cast<cudaStream_t>(stream);
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &early;
    cfg.numAttrs = pl.blocks > 0 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, norm_dw_kernel, (const float*)p.partial, pl.slots, d.n_col, dweight);
}

}  // namespace hx
