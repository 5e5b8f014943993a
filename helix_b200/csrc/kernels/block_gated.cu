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
// Bound by memory: every token is read once.  A CTA has 32 lanes' channels
// (4 bytes of a row per lane: 2 bf16 channels or 1 f32) of one chunk of 128
// tokens; warp w has kTok consecutive tokens of it, in registers.  (D, B) of
// the warps meet in shared memory, those of the CTAs of a cluster (cluster
// consecutive chunks of the same channels) in distributed shared memory, each
// CTA folds them onto the running state and the warps walk their tokens again
// from registers.  The cluster then moves on by its chunks, with the next
// chunk's loads already in flight.  Folds go in the order of the tokens:
// results do not depend on timing.
//
// The gradient walks the chunks from the end with c_t = f_t lam_t, the
// gradient that leaves token t for h_{t-1}: lam_t = dy_t + c_{t+1}, c_t =
// lam_t - z_t lam_t, so a run takes c to c - D c + E with the same D; h_{t-1}
// is walked forward again from the chunk's stored state.
#include <cooperative_groups.h>

#include "block_common.cuh"

namespace hx {
namespace {

namespace cg = cooperative_groups;

constexpr int kChunk = HELIX_GATED_CHUNK;
constexpr int kMaxCluster = 8;

// Channels per lane: 4 bytes of a row.
template <typename T>
struct Lane {
    static constexpr int kN = 4 / sizeof(T);
};

// z = 1 - sigmoid(g) and s = z (1 - z), both to a few ulp for every g: with
// t = e^-|g| and r = 1 / (1 + t), sigmoid(|g|) = r, sigmoid(-|g|) = t r.
// Subnormal t are kept: a gradient may scale them up again.
__device__ __forceinline__ void gate(float g, float& z, float& s) {
    float t;
    asm("ex2.approx.f32 %0, %1;" : "=f"(t) : "f"(-fabsf(g) * 1.4426950408889634f));
    const float r = __fdividef(1.0f, 1.0f + t);
    const float tr = t * r;
    z = g >= 0.0f ? tr : r;
    s = tr * r;
}

__device__ __forceinline__ float fold(float h, float d, float b) { return fmaf(-d, h, h) + b; }

// The lane's kN channels of a row, as raw bits; VEC: one 4-byte access.
template <typename T, bool VEC>
__device__ __forceinline__ uint32_t ld_raw(const T* p, int n) {
    if constexpr (sizeof(T) == 4) {
        return __ldcs(reinterpret_cast<const unsigned int*>(p));
    } else if (VEC && n == 2) {
        return __ldcs(reinterpret_cast<const unsigned int*>(p));
    } else {
        const unsigned short* q = reinterpret_cast<const unsigned short*>(p);
        const uint32_t lo = __ldcs(q), up = n == 2 ? __ldcs(q + 1) : 0;
        return lo | up << 16;
    }
}
template <typename T>
__device__ __forceinline__ void unpack(uint32_t w, float (&v)[Lane<T>::kN]) {
    if constexpr (sizeof(T) == 4) {
        v[0] = __uint_as_float(w);
    } else {
        v[0] = __uint_as_float(w << 16);
        v[1] = __uint_as_float(w & 0xffff0000u);
    }
}
template <typename T, bool VEC>
__device__ __forceinline__ void st_lane(T* p, int n, const float (&v)[Lane<T>::kN]) {
    if constexpr (sizeof(T) == 4) {
        __stcs(p, v[0]);
    } else if (VEC && n == 2) {
        __stcs(reinterpret_cast<unsigned int*>(p), bf16x2(v[0], v[1]));
    } else {
        p[0] = from_f32<T>(v[0]);
        if (n == 2) p[1] = from_f32<T>(v[1]);
    }
}

__device__ __forceinline__ int length_of(const GatedParams& p, int seq) {
    return p.lengths ? min(max(p.lengths[seq], 0), p.n_tok) : p.n_tok;
}

// The totals of the CTAs of a cluster, one step's and the next's.
template <int CB>
struct Totals {
    float d[2][kMaxCluster][CB], b[2][kMaxCluster][CB];
};

template <typename T, bool VEC, int kTok>
__global__ void __launch_bounds__(32 * (kChunk / kTok)) gated_kernel(const GatedParams p) {
    constexpr int N = Lane<T>::kN, CB = 32 * N, W = kChunk / kTok;
    __shared__ float agg_d[2][W][CB], agg_b[2][W][CB];
    __shared__ Totals<CB> tot;
    cg::cluster_group cluster = cg::this_cluster();

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int R = p.cluster, rank = (int)(blockIdx.x % (unsigned)R);
    const int slabs = (p.n_chan + CB - 1) / CB;
    const int slab = (int)(blockIdx.x / (unsigned)R) % slabs, seq = (int)(blockIdx.x / (unsigned)R) / slabs;
    const int c0 = slab * CB + N * lane;
    const int n = max(0, min(N, p.n_chan - c0));  // this lane's channels
    const int len = n > 0 ? length_of(p, seq) : 0;

    const T* g = static_cast<const T*>(p.g) + (int64_t)seq * p.seq_g + c0;
    const T* v = static_cast<const T*>(p.v) + (int64_t)seq * p.seq_v + c0;
    T* y = static_cast<T*>(p.y) + (int64_t)seq * p.seq_y + c0;

    float h[N];
#pragma unroll
    for (int e = 0; e < N; ++e) h[e] = p.h0 && e < n ? p.h0[(int64_t)seq * p.seq_h0 + c0 + e] : 0.0f;

    uint32_t gr[kTok], vr[kTok], vc[kTok];
    auto load = [&](int chunk) {
        const int t0 = chunk * kChunk + warp * kTok;
#pragma unroll
        for (int i = 0; i < kTok; ++i) {
            gr[i] = vr[i] = 0;
            if (t0 + i < len) {
                gr[i] = ld_raw<T, VEC>(g + (int64_t)(t0 + i) * p.s_g, n);
                vr[i] = ld_raw<T, VEC>(v + (int64_t)(t0 + i) * p.s_v, n);
            }
        }
    };
    const int steps = (p.n_chunk + R - 1) / R;
    if (steps > 0) load(rank);
    for (int s = 0; s < steps; ++s) {
        const int chunk = s * R + rank, buf = s & 1;
        const int t0 = chunk * kChunk + warp * kTok;
        float z[kTok][N], D[N], B[N];
#pragma unroll
        for (int e = 0; e < N; ++e) D[e] = B[e] = 0.0f;
#pragma unroll
        for (int i = 0; i < kTok; ++i) {
            float gv[N], vv[N];
            unpack<T>(gr[i], gv);
            unpack<T>(vr[i], vv);
            vc[i] = vr[i];
#pragma unroll
            for (int e = 0; e < N; ++e) {
                float slope;
                gate(gv[e], z[i][e], slope);
                if (t0 + i >= len) z[i][e] = 0.0f;
                D[e] = fmaf(z[i][e], 1.0f - D[e], D[e]);
                B[e] = fmaf(z[i][e], vv[e] - B[e], B[e]);
            }
        }
        if (s + 1 < steps) load(chunk + R);
#pragma unroll
        for (int e = 0; e < N; ++e) {
            agg_d[buf][warp][N * lane + e] = D[e];
            agg_b[buf][warp][N * lane + e] = B[e];
        }
        __syncthreads();
        // the CTA's totals, to every CTA of the cluster
        {
            const int c = (int)threadIdx.x % CB;
            float d = 0.0f, b = 0.0f;
#pragma unroll
            for (int w = 0; w < W; ++w) {
                const float dw = agg_d[buf][w][c];
                d = fmaf(dw, 1.0f - d, d);
                b = fold(b, dw, agg_b[buf][w][c]);
            }
            for (int k = (int)threadIdx.x / CB; k < R; k += 32 * W / CB) {
                Totals<CB>* to = cluster.map_shared_rank(&tot, k);
                to->d[buf][rank][c] = d;
                to->b[buf][rank][c] = b;
            }
        }
        if (R > 1)
            cluster.sync();
        else
            __syncthreads();
        float hw[N];  // the state entering this warp's tokens
#pragma unroll
        for (int e = 0; e < N; ++e) hw[e] = h[e];
        for (int k = 0; k < R; ++k) {
#pragma unroll
            for (int e = 0; e < N; ++e) {
                if (k == rank) hw[e] = h[e];
                h[e] = fold(h[e], tot.d[buf][k][N * lane + e], tot.b[buf][k][N * lane + e]);
            }
        }
        if (p.states && warp == 0 && chunk < p.n_chunk) {
            float* st = p.states + ((int64_t)seq * p.n_chunk + chunk) * p.n_chan + c0;
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (e < n) st[e] = hw[e];
        }
        for (int w = 0; w < warp; ++w)
#pragma unroll
            for (int e = 0; e < N; ++e)
                hw[e] = fold(hw[e], agg_d[buf][w][N * lane + e], agg_b[buf][w][N * lane + e]);
#pragma unroll
        for (int i = 0; i < kTok; ++i) {
            float vv[N], o[N];
            unpack<T>(vc[i], vv);
#pragma unroll
            for (int e = 0; e < N; ++e) {
                hw[e] = fmaf(z[i][e], vv[e] - hw[e], hw[e]);
                o[e] = t0 + i < len ? hw[e] : 0.0f;
            }
            if (t0 + i < p.n_tok && n > 0) st_lane<T, VEC>(y + (int64_t)(t0 + i) * p.s_y, n, o);
        }
    }
    // every CTA holds the last state; in place of h0 is safe because each has
    // read h0 before the cluster's first barrier
    if (rank == 0 && warp == 0) {
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (e < n) p.h1[(int64_t)seq * p.seq_h1 + c0 + e] = h[e];
    }
    if (R > 1) cluster.sync();  // no CTA leaves while another may write its totals
}

template <typename T, bool VEC, int kTok>
__global__ void __launch_bounds__(32 * (kChunk / kTok)) gated_grad_kernel(const GatedParams p) {
    constexpr int N = Lane<T>::kN, CB = 32 * N, W = kChunk / kTok;
    __shared__ float agg_d[W][CB], agg_b[W][CB], agg_e[W][CB];
    __shared__ Totals<CB> tot;
    cg::cluster_group cluster = cg::this_cluster();

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int R = p.cluster, rank = (int)(blockIdx.x % (unsigned)R);
    const int slabs = (p.n_chan + CB - 1) / CB;
    const int slab = (int)(blockIdx.x / (unsigned)R) % slabs, seq = (int)(blockIdx.x / (unsigned)R) / slabs;
    const int c0 = slab * CB + N * lane;
    const int n = max(0, min(N, p.n_chan - c0));
    const int len = n > 0 ? length_of(p, seq) : 0;

    const T* g = static_cast<const T*>(p.g) + (int64_t)seq * p.seq_g + c0;
    const T* v = static_cast<const T*>(p.v) + (int64_t)seq * p.seq_v + c0;
    const T* dy = static_cast<const T*>(p.dy) + (int64_t)seq * p.seq_dy + c0;
    T* dv = static_cast<T*>(p.dv) + (int64_t)seq * p.seq_dv + c0;
    T* dg = static_cast<T*>(p.dg) + (int64_t)seq * p.seq_dg + c0;

    float c[N];  // the gradient entering the step's tokens from behind
#pragma unroll
    for (int e = 0; e < N; ++e) c[e] = p.dh1 && e < n ? p.dh1[(int64_t)seq * p.seq_dh1 + c0 + e] : 0.0f;

    uint32_t gr[kTok], vr[kTok], yr[kTok];
    auto load = [&](int chunk) {
        const int t0 = chunk * kChunk + warp * kTok;
#pragma unroll
        for (int i = 0; i < kTok; ++i) {
            gr[i] = vr[i] = yr[i] = 0;
            if (t0 + i < len) {
                gr[i] = ld_raw<T, VEC>(g + (int64_t)(t0 + i) * p.s_g, n);
                vr[i] = ld_raw<T, VEC>(v + (int64_t)(t0 + i) * p.s_v, n);
                yr[i] = ld_raw<T, VEC>(dy + (int64_t)(t0 + i) * p.s_dy, n);
            }
        }
    };
    const int steps = (p.n_chunk + R - 1) / R;
    if (steps > 0) load((steps - 1) * R + rank);
    for (int s = steps - 1; s >= 0; --s) {
        const int chunk = s * R + rank, buf = s & 1;
        const int t0 = chunk * kChunk + warp * kTok;
        float z[kTok][N], q[kTok][N], D[N], B[N], E[N];
        uint32_t yc[kTok], vc[kTok];
        float hw[N];
#pragma unroll
        for (int e = 0; e < N; ++e) {
            D[e] = B[e] = E[e] = 0.0f;
            hw[e] = e < n && chunk < p.n_chunk
                        ? p.states[((int64_t)seq * p.n_chunk + chunk) * p.n_chan + c0 + e] : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < kTok; ++i) {
            float gv[N], vv[N];
            unpack<T>(gr[i], gv);
            unpack<T>(vr[i], vv);
            vc[i] = vr[i];
            yc[i] = yr[i];
#pragma unroll
            for (int e = 0; e < N; ++e) {
                gate(gv[e], z[i][e], q[i][e]);
                if (t0 + i >= len) z[i][e] = q[i][e] = 0.0f;
                D[e] = fmaf(z[i][e], 1.0f - D[e], D[e]);
                B[e] = fmaf(z[i][e], vv[e] - B[e], B[e]);
            }
        }
#pragma unroll
        for (int i = kTok - 1; i >= 0; --i) {
            float dd[N];
            unpack<T>(yc[i], dd);
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const float lam = dd[e] + E[e];
                E[e] = fmaf(-z[i][e], lam, lam);
            }
        }
        if (s > 0) load(chunk - R);
#pragma unroll
        for (int e = 0; e < N; ++e) {
            agg_d[warp][N * lane + e] = D[e];
            agg_b[warp][N * lane + e] = B[e];
            agg_e[warp][N * lane + e] = E[e];
        }
        __syncthreads();
        {
            const int ch = (int)threadIdx.x % CB;
            float d = 0.0f, b = 0.0f;
#pragma unroll
            for (int w = W - 1; w >= 0; --w) {
                const float dw = agg_d[w][ch];
                d = fmaf(dw, 1.0f - d, d);
                b = fold(b, dw, agg_e[w][ch]);
            }
            for (int k = (int)threadIdx.x / CB; k < R; k += 32 * W / CB) {
                Totals<CB>* to = cluster.map_shared_rank(&tot, k);
                to->d[buf][rank][ch] = d;
                to->b[buf][rank][ch] = b;
            }
        }
        // the warp's entry state and what it makes of h_{t-1} - v_t
        for (int w = 0; w < warp; ++w)
#pragma unroll
            for (int e = 0; e < N; ++e)
                hw[e] = fold(hw[e], agg_d[w][N * lane + e], agg_b[w][N * lane + e]);
#pragma unroll
        for (int i = 0; i < kTok; ++i) {
            float vv[N];
            unpack<T>(vc[i], vv);
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const float off = hw[e] - vv[e];
                q[i][e] *= off;
                hw[e] = fmaf(-z[i][e], off, hw[e]);
            }
        }
        if (R > 1)
            cluster.sync();
        else
            __syncthreads();
        float cw[N];
#pragma unroll
        for (int e = 0; e < N; ++e) cw[e] = c[e];
        for (int k = R - 1; k >= 0; --k) {
#pragma unroll
            for (int e = 0; e < N; ++e) {
                if (k == rank) cw[e] = c[e];
                c[e] = fold(c[e], tot.d[buf][k][N * lane + e], tot.b[buf][k][N * lane + e]);
            }
        }
        for (int w = W - 1; w > warp; --w)
#pragma unroll
            for (int e = 0; e < N; ++e)
                cw[e] = fold(cw[e], agg_d[w][N * lane + e], agg_e[w][N * lane + e]);
#pragma unroll
        for (int i = kTok - 1; i >= 0; --i) {
            float dd[N], ov[N], og[N];
            unpack<T>(yc[i], dd);
            const bool live = t0 + i < len;
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const float lam = dd[e] + cw[e];
                const float zl = z[i][e] * lam;
                ov[e] = live ? zl : 0.0f;
                og[e] = live ? lam * q[i][e] : 0.0f;
                cw[e] = lam - zl;
            }
            if (t0 + i < p.n_tok && n > 0) {
                st_lane<T, VEC>(dv + (int64_t)(t0 + i) * p.s_dv, n, ov);
                st_lane<T, VEC>(dg + (int64_t)(t0 + i) * p.s_dg, n, og);
            }
        }
        __syncthreads();  // the warps' shares are read before the next step writes them
    }
    if (p.dh0 && rank == 0 && warp == 0) {
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (e < n) p.dh0[(int64_t)seq * p.seq_dh0 + c0 + e] = c[e];
    }
    if (R > 1) cluster.sync();
}

int launch_clusters(void (*kernel)(GatedParams), const GatedParams& p, int64_t groups, int threads, void* stream) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(groups * p.cluster));
    cfg.blockDim = dim3((unsigned)threads);
    cfg.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = (unsigned)p.cluster;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, p);
}

// CTAs of a cluster: as many chunks in flight as fill the GPU twice over.
int cluster_of(const helix_ctx* ctx, int64_t groups, int chunks) {
    int r = 1;
    while (r < kMaxCluster && r < chunks && groups * r < 4 * (int64_t)ctx->n_sm) r *= 2;
    return r;
}

template <typename T, bool VEC>
int launch_gated_t(const helix_ctx* ctx, GatedParams p, bool grad, void* stream) {
    constexpr int CB = 32 * Lane<T>::kN;
    const int64_t groups = (int64_t)p.n_seq * ((p.n_chan + CB - 1) / CB);
    p.cluster = cluster_of(ctx, groups, p.n_chunk);
    if (grad) return launch_clusters(gated_grad_kernel<T, VEC, 8>, p, groups, 32 * kChunk / 8, stream);
    return launch_clusters(gated_kernel<T, VEC, 16>, p, groups, 32 * kChunk / 16, stream);
}

int launch_gated_any(const helix_ctx* ctx, const helix_gated_scan_desc& d, const GatedParams& p, bool vec, bool grad,
                     void* stream) {
    if (d.io_dtype == HELIX_F32) return launch_gated_t<float, true>(ctx, p, grad, stream);
    return vec ? launch_gated_t<__nv_bfloat16, true>(ctx, p, grad, stream)
               : launch_gated_t<__nv_bfloat16, false>(ctx, p, grad, stream);
}

}  // namespace

int launch_gated(const helix_ctx* ctx, const helix_gated_scan_desc& d, GatedParams p, bool vec, void* stream) {
    return launch_gated_any(ctx, d, p, vec, false, stream);
}

int launch_gated_grad(const helix_ctx* ctx, const helix_gated_scan_desc& d, GatedParams p, bool vec, void* stream) {
    return launch_gated_any(ctx, d, p, vec, true, stream);
}

}  // namespace hx
