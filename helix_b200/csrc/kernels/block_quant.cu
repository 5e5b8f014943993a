// block_quant.cu -- a matrix in 8 bits with one scale per 128 columns of a
// row or per 128 x 128 block, as it is or transposed.
//
// Bound by memory: 2 or 4 bytes read and 1 written per value, one pass.  A
// CTA holds a 128 x 128 tile in registers: half-warp (w, hi) has rows
// 16 w + 8 hi .. + 7, a lane 8 columns of each, so that a lane's 8 x 8 values
// turn into 8 bytes of each of 8 rows of the transposed output.  Transposed
// tiles pass through shared memory (16 KB, 8-byte units swizzled so that
// neither side has bank conflicts) to leave as whole 128-byte rows.
//
// Measured: 8192 x 4096 bf16 (15.4 us at the measured copy rate) by blocks 16.8
// us, by rows 20.1, transposed by rows 22.2, where every tile waits at two
// barriers for its columns' largest values; 8192 x 4095, rows at odd addresses,
// 28.5 by rows.
#include "block_common.cuh"
#include "umma.cuh"

namespace hx {
namespace {

constexpr int kTile = HELIX_GROUP;
constexpr int kQThreads = 256;

__device__ __forceinline__ int unit_of(int col, int unit) { return unit ^ (((col >> 3) ^ col) & 15); }

// Eight consecutive values at any address of the type's alignment: the
// aligned 16-byte pieces that hold those before `end` (zeros for the others),
// and the values shifted out of them.  Every piece read holds a value that
// exists.
template <typename T>
struct Any8 {
    static constexpr int kPieces = (int)sizeof(T) / 2 + 1;
    uint32_t w[4 * kPieces], off;
    __device__ __forceinline__ void load(const T* p, const T* end) {
        const uintptr_t at = reinterpret_cast<uintptr_t>(p), to = reinterpret_cast<uintptr_t>(end);
        off = (uint32_t)(at & 15);
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const uintptr_t q = at - off + 16 * i;
            uint4 v = make_uint4(0u, 0u, 0u, 0u);
            if (at < to && q < to && (i < kPieces - 1 || off)) v = *reinterpret_cast<const uint4*>(q);
            w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
        }
    }
    __device__ __forceinline__ void get(float (&f)[8]) {
#pragma unroll
        for (int i = 0; i + 2 < 4 * kPieces; ++i) w[i] = off & 8 ? w[i + 2] : w[i];
#pragma unroll
        for (int i = 0; i + 3 < 4 * kPieces; ++i) w[i] = off & 4 ? w[i + 1] : w[i];
        if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = off & 2 ? __funnelshift_r(w[i], w[i + 1], 16) : w[i];
        }
        Raw8<T> raw;
#pragma unroll
        for (int i = 0; i < kPieces - 1; ++i)
            raw.v[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
        raw.unpack(f);
    }
};

// Both times `by`, in one instruction (8192 x 4096 bf16 by rows: 21.7 -> 20.1
// us; not where the pair would be of two rows: 22.2 -> 23.0).
__device__ __forceinline__ void mul2(float& a, float& b, float by) {
    umma::f2_to(umma::f2_mul(umma::f2_of(a, b), umma::f2_of(by, by)), a, b);
}

template <typename T, bool BLOCKS, bool TURN, bool VEC>
__global__ void __launch_bounds__(kQThreads, 3) quant_kernel(const QuantParams p) {
    __shared__ __align__(16) uint8_t turned[TURN ? kTile * kTile : 16];
    __shared__ float peak[8][TURN && !BLOCKS ? kTile : 1];
    __shared__ float col_scale[TURN && !BLOCKS ? kTile : 1];

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, hi = lane >> 4, l = lane & 15;
    const int64_t r0 = (int64_t)(blockIdx.x / p.n_tile_col) * kTile;
    const int64_t c0 = (int64_t)(blockIdx.x % p.n_tile_col) * kTile;
    const int rows = (int)(p.n_row - r0 < kTile ? p.n_row - r0 : kTile);
    const int cols = (int)(p.n_col - c0 < kTile ? p.n_col - c0 : kTile);
    const int rt = 16 * warp + 8 * hi;  // the lane's first row
    auto col = [&](int e) { return 8 * l + e; };

    float x[8][8];
    const T* src = static_cast<const T*>(p.x) + r0 * p.ld_x + c0;
    // every load of a row (misaligned: of half the rows) before the first look
    if constexpr (VEC) {
        Raw8<T> raw[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            raw[i].zero();
            if (rt + i < rows && 8 * l + 8 <= cols) raw[i].load(src + (int64_t)(rt + i) * p.ld_x + 8 * l);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) raw[i].unpack(x[i]);
        if (8 * l < cols && 8 * l + 8 > cols) {  // a row's last values where they are no whole eight
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int e = 0; e < 7; ++e)
                    if (rt + i < rows && col(e) < cols) x[i][e] = to_f32(src[(int64_t)(rt + i) * p.ld_x + col(e)]);
        }
    } else {
#pragma unroll
        for (int h = 0; h < 8; h += 4) {
            Any8<T> any[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const T* row = src + (int64_t)(rt + h + i) * p.ld_x;
                any[i].load(row + 8 * l, row + (rt + h + i < rows ? cols : 0));
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                any[i].get(x[h + i]);
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (col(e) >= cols) x[h + i][e] = 0.0f;
            }
        }
    }

    // every value becomes value / scale
    if constexpr (BLOCKS) {
        float a = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int e = 0; e < 8; e += 2) a = max_abs_nan(a, x[i][e], x[i][e + 1]);
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) a = max_nan(a, __shfl_xor_sync(0xffffffffu, a, o));
        if (lane == 0) peak[warp][0] = a;
        __syncthreads();
        a = peak[0][0];
#pragma unroll
        for (int w = 1; w < 8; ++w) a = max_nan(a, peak[w][0]);
        float inv;
        const float scale = group_scale(a, &inv);
        if (threadIdx.x == 0)
            p.scale[(TURN ? c0 / kTile : r0 / kTile) * p.ld_scale + (TURN ? r0 / kTile : c0 / kTile)] = scale;
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int e = 0; e < 8; e += 2) mul2(x[i][e], x[i][e + 1], inv);
    } else if constexpr (!TURN) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float a = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; e += 2) a = max_abs_nan(a, x[i][e], x[i][e + 1]);
#pragma unroll
            for (int o = 8; o >= 1; o >>= 1) a = max_nan(a, __shfl_xor_sync(0xffffffffu, a, o));
            float inv;
            const float scale = group_scale(a, &inv);
            if (l == 0 && rt + i < rows) p.scale[(r0 + rt + i) * p.ld_scale + c0 / kTile] = scale;
#pragma unroll
            for (int e = 0; e < 8; e += 2) mul2(x[i][e], x[i][e + 1], inv);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            float a = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; i += 2) a = max_abs_nan(a, x[i][e], x[i + 1][e]);
            a = max_nan(a, __shfl_xor_sync(0xffffffffu, a, 16));
            if (hi == 0) peak[warp][col(e)] = a;
        }
        __syncthreads();
        if (threadIdx.x < kTile) {
            const int c = threadIdx.x;
            float a = peak[0][c];
#pragma unroll
            for (int w = 1; w < 8; ++w) a = max_nan(a, peak[w][c]);
            const float scale = group_scale(a, &col_scale[c]);
            if (c < cols) p.scale[(c0 + c) * p.ld_scale + r0 / kTile] = scale;
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float inv = col_scale[col(e)];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i][e] *= inv;
        }
    }

    if constexpr (!TURN) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (rt + i >= rows) break;
            uint8_t* q = p.q + (r0 + rt + i) * p.ld_q + c0;
            if (p.q_vec && 8 * l + 8 <= cols) {
                *reinterpret_cast<uint2*>(q + 8 * l) =
                    make_uint2(e4m3x2(x[i][0], x[i][1]) | e4m3x2(x[i][2], x[i][3]) << 16,
                               e4m3x2(x[i][4], x[i][5]) | e4m3x2(x[i][6], x[i][7]) << 16);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (col(e) < cols) q[col(e)] = (uint8_t)e4m3x2(x[i][e], 0.0f);
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            *reinterpret_cast<uint2*>(turned + col(e) * kTile + 8 * unit_of(col(e), rt >> 3)) =
                make_uint2(e4m3x2(x[0][e], x[1][e]) | e4m3x2(x[2][e], x[3][e]) << 16,
                           e4m3x2(x[4][e], x[5][e]) | e4m3x2(x[6][e], x[7][e]) << 16);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int c = 16 * i + 2 * warp + hi;  // row of q, unit l of it
            if (c >= cols) continue;
            const uint2 v = *reinterpret_cast<const uint2*>(turned + c * kTile + 8 * unit_of(c, l));
            uint8_t* q = p.q + (c0 + c) * p.ld_q + r0 + 8 * l;
            if (p.q_vec && 8 * l + 8 <= rows) {
                *reinterpret_cast<uint2*>(q) = v;
            } else {
#pragma unroll
                for (int b = 0; b < 8; ++b)
                    if (8 * l + b < rows) q[b] = (uint8_t)((b < 4 ? v.x >> (8 * b) : v.y >> (8 * (b - 4))) & 0xff);
            }
        }
    }
}

template <typename T, bool VEC>
int launch_quant_t(const helix_quant8_desc& d, const QuantParams& p, dim3 grid, void* stream) {
    if (d.form == HELIX_SCALE_BLOCKS)
        return d.transpose ? block_launch(quant_kernel<T, true, true, VEC>, grid, dim3(kQThreads), 0, stream, p)
                           : block_launch(quant_kernel<T, true, false, VEC>, grid, dim3(kQThreads), 0, stream, p);
    return d.transpose ? block_launch(quant_kernel<T, false, true, VEC>, grid, dim3(kQThreads), 0, stream, p)
                       : block_launch(quant_kernel<T, false, false, VEC>, grid, dim3(kQThreads), 0, stream, p);
}

}  // namespace

int launch_quant(const helix_quant8_desc& d, const QuantParams& p, bool vec, void* stream) {
    const dim3 grid((unsigned)((d.n_row + kTile - 1) / kTile * p.n_tile_col));
    if (d.x_dtype == HELIX_F32)
        return vec ? launch_quant_t<float, true>(d, p, grid, stream) : launch_quant_t<float, false>(d, p, grid, stream);
    return vec ? launch_quant_t<__nv_bfloat16, true>(d, p, grid, stream)
               : launch_quant_t<__nv_bfloat16, false>(d, p, grid, stream);
}

}  // namespace hx
