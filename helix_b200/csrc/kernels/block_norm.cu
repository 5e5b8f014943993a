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
// Sums, statistics and the products are fp32; the only roundings are those
// of the stored sum, the output and (8 bits) 1 / scale.
//
// Measured: 8192 x 4096 bf16 to 8 bits 45 us, 5.2 TB/s; 1537 x 2501 f32 10.9,
// 5.6; 4096 x 16384 bf16 111; gradient of 16384 x 4096 bf16 113, 4.8 TB/s.  A
// copy reaches 6.6 at sizes where a launch's start and end do not count.  What
// the norm lacks is the wait of a row for its statistic, which the SM's other
// rows cover in part; the gradient also reads the weights from L1 for each row.
#include <algorithm>

#include "block_common.cuh"

namespace hx {
namespace {

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
    __device__ __forceinline__ void get(const T* row, int c0, int lane, int n_col, float (&v)[8]) const {
        if constexpr (VEC) {
            raw.unpack(v);
            // a row's last values where they are no whole eight
            const int c = c0 + 8 * lane;
            if (c < n_col && c + 8 > n_col) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (c + e < n_col) v[e] = to_f32(row[c + e]);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = to_f32(one[e]);
        }
    }
};
template <bool VEC, typename T>
__device__ __forceinline__ void st_seg(T* row, int c0, int lane, int n_col, const float (&v)[8]) {
    if (VEC && c0 + 8 * lane + 8 <= n_col) {
        st8(row + c0 + 8 * lane, v);
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int c = col_of<VEC>(c0, lane, e);
        if (c < n_col) row[c] = from_f32<T>(v[e]);
    }
}
template <bool VEC, typename T>
__device__ __forceinline__ void ld_seg(const T* row, int c0, int lane, int n_col, float (&v)[8]) {
    Seg<VEC, T> s;
    s.load(row, c0, lane, n_col);
    s.get(row, c0, lane, n_col, v);
}
template <bool VEC>
__device__ __forceinline__ void ld_weight(const NormParams& p, int c0, int lane, float (&v)[8]) {
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

// Sum over the wpr warps of a row (every warp of the block calls it).
// `part` holds one float per warp; buffers alternate between calls so that
// one barrier a call is enough.
__device__ __forceinline__ float row_sum(float v, int wpr, int warp, int lane, float* part) {
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (wpr == 1) return v;
    if (lane == 0) part[warp] = v;
    __syncthreads();
    const int first = warp / wpr * wpr;
    float s = 0.0f;
    for (int w = 0; w < wpr; ++w) s += part[first + w];
    return s;
}

// The segment's 8 values a lane holds, as e4m3 with its group's scale.
template <bool VEC>
__device__ __forceinline__ void st_seg_e4m3(const NormParams& p, int64_t row, int c0, int lane,
                                            const float (&n)[8]) {
    uint8_t* q = static_cast<uint8_t*>(p.out) + row * p.ld_out;
    float* sc = p.scale + row * p.ld_scale;
    if constexpr (VEC) {
        float a = fabsf(n[0]);
#pragma unroll
        for (int e = 1; e < 8; ++e) a = max_nan(a, fabsf(n[e]));
#pragma unroll
        for (int o = 8; o >= 1; o >>= 1) a = max_nan(a, __shfl_xor_sync(0xffffffffu, a, o));
        float inv;
        const float scale = group_scale(a, &inv);
        const int c = c0 + 8 * lane;
        if ((lane & 15) == 0 && c < p.n_col) sc[c / HELIX_GROUP] = scale;
        if (c + 8 <= p.n_col) {
            *reinterpret_cast<uint2*>(q + c) =
                make_uint2(e4m3x2(n[0] * inv, n[1] * inv) | e4m3x2(n[2] * inv, n[3] * inv) << 16,
                           e4m3x2(n[4] * inv, n[5] * inv) | e4m3x2(n[6] * inv, n[7] * inv) << 16);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (c + e < p.n_col) q[c + e] = (uint8_t)e4m3x2(n[e] * inv, 0.0f);
        }
    } else {
#pragma unroll
        for (int g = 0; g < 2; ++g) {  // the segment's groups: e = 0..3 and 4..7
            float a = 0.0f;
#pragma unroll
            for (int e = 4 * g; e < 4 * g + 4; ++e) a = max_nan(a, fabsf(n[e]));
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

    float s[V][8];
    float ss = 0.0f;
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
            float v[8];
            sx[j].get(x, c0, lane, n, s[j]);
            sr[j].get(r, c0, lane, p.res ? n : 0, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if (p.res) s[j][e] += v[e];
                ss += s[j][e] * s[j][e];
            }
        }
    }
    ss = row_sum(ss, p.wpr, warp, lane, part);
    if (!live) return;
    const float rstd = 1.0f / sqrtf(ss / (float)p.n_col + p.eps);
    if (p.rstd && wr == 0 && lane == 0) p.rstd[row] = rstd;

#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int c0 = (j * p.wpr + wr) * kSeg;
        if (p.sum) st_seg<VEC>(static_cast<TR*>(p.sum) + row * p.ld_sum, c0, lane, p.n_col, s[j]);
        float w[8];
        ld_weight<VEC>(p, c0, lane, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] *= s[j][e] * rstd;
        if (p.out_dtype == HELIX_E4M3)
            st_seg_e4m3<VEC>(p, row, c0, lane, w);
        else if (p.out_dtype == HELIX_BF16)
            st_seg<VEC>(static_cast<__nv_bfloat16*>(p.out) + row * p.ld_out, c0, lane, p.n_col, w);
        else
            st_seg<VEC>(static_cast<float*>(p.out) + row * p.ld_out, c0, lane, p.n_col, w);
    }
}

// 48 registers, so that five blocks fit an SM (8192 x 4096 bf16: 45 us, with
// four 49).
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

// Persistent: a row slot takes every slots-th row and keeps its share of
// dweight in registers, written to partial[slot] at the end.
template <typename TX, typename TR, int V, bool VEC>
__global__ void __launch_bounds__(V == 1 ? 1024 : 512, 1) norm_grad_kernel(const NormParams p) {
    __shared__ float part[2][kMaxWarps];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rg = warp / p.wpr, wr = warp % p.wpr;
    // The widest rows (V = 4) leave no registers for dweight, which then stays
    // in shared memory, nor for loads ahead.
    constexpr bool kWide = V == 4;
    extern __shared__ float dw_smem[];
    float dw[kWide ? 1 : V][8];
    auto dw_at = [&](int j, int e) -> float& {
        if constexpr (kWide)
            return dw_smem[(8 * j + e) * blockDim.x + threadIdx.x];
        else
            return dw[j][e];
    };
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) dw_at(j, e) = 0.0f;

    // a row's loads are in flight while the row before is worked on
    Seg<VEC, TX> sd[V];
    Seg<VEC, TR> ss[V], sa[V];
    float rstd_next = 0.0f;
    const TX* dout = static_cast<const TX*>(p.dout);
    const TR* sum = static_cast<const TR*>(p.sum);
    const TR* dsum = static_cast<const TR*>(p.dsum);
    auto fetch = [&](int64_t row) {
        const int n = row < p.n_row ? p.n_col : 0;
        row = n ? row : 0;
        rstd_next = n ? p.rstd[row] : 0.0f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int c0 = (j * p.wpr + wr) * kSeg;
            sd[j].load(dout + row * p.ld_dout, c0, lane, n);
            ss[j].load(sum + row * p.ld_sum, c0, lane, n);
            if (!kWide) sa[j].load(dsum + row * p.ld_dsum, c0, lane, p.dsum ? n : 0);
        }
    };

    int turn = 0;
    const int64_t step = (int64_t)gridDim.x * p.rpb;
    if (!kWide) fetch((int64_t)blockIdx.x * p.rpb + rg);
    for (int64_t base = (int64_t)blockIdx.x * p.rpb; base < p.n_row; base += step) {
        const bool live = base + rg < p.n_row;
        const int64_t row = live ? base + rg : 0;
        const int n = live ? p.n_col : 0;
        if (kWide) {
            fetch(base + rg);
            if (base + step < p.n_row) {  // the next row goes to L2
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const int c0 = (j * p.wpr + wr) * kSeg;
                    prefetch_seg(dout + (base + step) * p.ld_dout, c0, lane, p.n_col);
                    prefetch_seg(sum + (base + step) * p.ld_sum, c0, lane, p.n_col);
                    if (p.dsum) prefetch_seg(dsum + (base + step) * p.ld_dsum, c0, lane, p.n_col);
                }
            }
        }
        const float rstd = rstd_next;
        float d[V][8], s[V][8], o[kWide ? 1 : V][8];
        float along = 0.0f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int c0 = (j * p.wpr + wr) * kSeg;
            float w[8];
            sd[j].get(dout + row * p.ld_dout, c0, lane, n, d[j]);
            ss[j].get(sum + row * p.ld_sum, c0, lane, n, s[j]);
            if constexpr (!kWide) sa[j].get(dsum + row * p.ld_dsum, c0, lane, p.dsum ? n : 0, o[j]);
            ld_weight<VEC>(p, c0, lane, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                s[j][e] *= rstd;              // s rstd
                dw_at(j, e) += d[j][e] * s[j][e];
                d[j][e] *= w[e];              // dn w
                along += d[j][e] * s[j][e];
            }
        }
        if (!kWide) fetch(base + step + rg);
        along = row_sum(along, p.wpr, warp, lane, part[turn]) / (float)p.n_col;
        turn ^= 1;
        if (!live) continue;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int c0 = (j * p.wpr + wr) * kSeg;
            float(&v)[8] = o[kWide ? 0 : j];
            if constexpr (kWide) ld_seg<VEC>(dsum + row * p.ld_dsum, c0, lane, p.dsum ? n : 0, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += rstd * (d[j][e] - s[j][e] * along);
            st_seg<VEC>(static_cast<TX*>(p.dx) + row * p.ld_dx, c0, lane, n, v);
            if (p.dres) st_seg<VEC>(static_cast<TR*>(p.dres) + row * p.ld_dres, c0, lane, n, v);
        }
    }
    float* mine = p.partial + ((int64_t)blockIdx.x * p.rpb + rg) * p.n_col;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int c0 = (j * p.wpr + wr) * kSeg;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int c = col_of<VEC>(c0, lane, e);
            if (c < p.n_col) mine[c] = dw_at(j, e);
        }
    }
}

// dweight[c] = the partials' sum in the order of the slots.
constexpr int kDwRows = 16;
__global__ void __launch_bounds__(32 * kDwRows) norm_dw_kernel(const float* partial, int slots, int n_col,
                                                              float* dweight) {
    __shared__ float part[kDwRows][33];
    const int lane = threadIdx.x & 31, r = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + lane;
    float v = 0.0f;
    if (c < n_col)
#pragma unroll 8
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
        return v == 1   ? block_launch(norm_grad_kernel<TX, TR, 1, VEC>, grid, block, 0, stream, p)
               : v == 2 ? block_launch(norm_grad_kernel<TX, TR, 2, VEC>, grid, block, 0, stream, p)
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

template <typename TX, typename TR>
int configure_norm_t() {
    const int e = cudaFuncSetAttribute(norm_grad_kernel<TX, TR, 4, true>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       (int)kWideSmem);
    if (e != cudaSuccess) return e;
    return cudaFuncSetAttribute(norm_grad_kernel<TX, TR, 4, false>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                (int)kWideSmem);
}

}  // namespace

int configure_norm() {
    int e;
    if ((e = configure_norm_t<float, float>()) != cudaSuccess) return e;
    if ((e = configure_norm_t<__nv_bfloat16, float>()) != cudaSuccess) return e;
    return configure_norm_t<__nv_bfloat16, __nv_bfloat16>();
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

// The gradient holds two rows, a third on its way, and dweight.  One segment
// per warp leaves 64 registers enough (16384 x 4096 bf16: 113 us, with two 142);
// single accesses need twice the registers, and two segments (8192 x 4095: 99
// us, with one 163); the widest rows have four.
NormGradPlan norm_grad_plan(const helix_ctx* ctx, const helix_rms_norm_desc& d, bool vec) {
    NormGradPlan pl{};
    const int segs = (d.n_col + kSeg - 1) / kSeg;
    pl.shape = shape_of(d.n_col, segs > 32 ? 4 : vec || segs == 1 ? 1 : 2);
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
    return block_launch(norm_dw_kernel, dim3((unsigned)((d.n_col + 31) / 32)), dim3(32 * kDwRows), 0, stream,
                        (const float*)p.partial, pl.slots, d.n_col, dweight);
}

}  // namespace hx
