// Layer norm over the rows of x [M, D], forward and backward, with the reduction of the weight's and the bias's gradient.
//
//   mu = mean x,  r = 1 / sqrt(mean (x - mu)^2 + eps),  h = (x - mu) r,  y = w h + b
//   dx = r (w g - mean(w g) - h mean(w g h))  [* LeakyReLU'(x): x a LeakyReLU's output],   dw = sum_m g h,   db = sum_m g
//
// Both directions read every operand once and keep the row in registers between the passes over it (the variance is taken about the
// mean, not from a difference of moments); statistics and sums are fp32.  TPR neighbouring threads own a row, each holds NV pieces of
// 16 bytes of it (8 lanes to 16 waves; rule: plan()).  Any of the row types fp32 / bf16 / fp16, any width up to 16384, any row
// stride.  The forward optionally also writes the row's 8-bit form (act8.h), and the backward takes x from it: the norm's saved input
// is then one byte per value, and LeakyReLU' reads off its codes.
//
// The backward's column sums: a thread owns columns, so dw and db accumulate in its registers over all rows of its workgroup; the
// workgroups' partial rows [G, 2, D] are joined in workgroup order by a second kernel (no atomics: the same bits every run).
#include "act8.h"

using namespace pcvae;

namespace {

constexpr int kMaxWidth = 16384;
constexpr int kBwdGroups = 512;   // workgroups of a backward launch at most: two per CU, and so many partial rows to join

struct FwdParams {
    const void* x; int64_t ldx;
    const float* w; const float* b;
    void* y; int64_t ldy;
    float* mean; float* rstd;
    uint8_t* codes; int64_t ldc; uint8_t* scales; int64_t lds;
    int64_t M; int D, Dp;
    float eps;
};
struct BwdParams {
    const void* g; int64_t ldg;
    const void* x; int64_t ldx;
    const uint8_t* codes; int64_t ldc; const uint8_t* scales; int64_t lds;
    const float* w; const float* mean; const float* rstd;
    void* dx; int64_t lddx;
    float* part;
    int64_t M; int D, Dp;
    int leaky;
    float inv_d;
};

// sums of N values over the TPR threads of a row, every thread gets them.  Rows of more than a wave go through LDS; `slot` alternates
// between two consecutive calls, so a wave that is ahead writes the slot the others have left behind at the barrier between.
template <int TPR, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float (*red)[N][16], int slot) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = lanes_sum<(TPR < 64 ? TPR : 64)>(v[i]);
    if constexpr (TPR > 64) {
        constexpr int W = TPR / 64;
        const int wave = threadIdx.x / 64;
        if ((threadIdx.x & 63) == 0) {
#pragma unroll
            for (int i = 0; i < N; ++i) red[slot][i][wave] = v[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float s = 0.f;
#pragma unroll
            for (int k = 0; k < W; ++k) s += red[slot][i][k];
            v[i] = s;
        }
    }
}

template <typename T, int TPR, int NV, bool KEEP>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void layer_norm_fwd_kernel(FwdParams p) {
    constexpr int BLOCK = TPR > 256 ? TPR : 256, ROWS = BLOCK / TPR, VW = RowType<T>::VW;
    __shared__ float red0[2][1][16], red1[2][2][16];
    const int lane = threadIdx.x % TPR, sub = threadIdx.x / TPR;
    float w[NV][VW], b[NV][VW];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int c = (k * TPR + lane) * VW;
#pragma unroll
        for (int i = 0; i < VW; ++i) {
            w[k][i] = p.w && c + i < p.D ? p.w[c + i] : 1.f;
            b[k][i] = p.b && c + i < p.D ? p.b[c + i] : 0.f;
        }
    }
    for (int64_t row0 = (int64_t)blockIdx.x * ROWS; row0 < p.M; row0 += (int64_t)gridDim.x * ROWS) {
        const bool live = row0 + sub < p.M;
        const int64_t row = live ? row0 + sub : p.M - 1;
        const T* xr = static_cast<const T*>(p.x) + row * p.ldx;
        float v[NV][VW], s[1] = {0.f};
#pragma unroll
        for (int k = 0; k < NV; ++k) load_cols(xr, (k * TPR + lane) * VW, p.D, v[k]);
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int i = 0; i < VW; ++i) s[0] += v[k][i];
        row_sum<TPR, 1>(s, red0, 0);
        const float near = s[0] / p.D;
        float m[2] = {0.f, 0.f};
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = (k * TPR + lane) * VW;
#pragma unroll
            for (int i = 0; i < VW; ++i) {
                const float d = c + i < p.D ? v[k][i] - near : 0.f;
                m[0] += d;
                m[1] = fmaf(d, d, m[1]);
            }
        }
        // what the first sum's roundings left of the mean shows in the deviations' own mean: rows far from zero (and constant ones) need it
        row_sum<TPR, 2>(m, red1, 0);
        const float rest = m[0] / p.D, mean = near + rest;
        const float rstd = 1.f / sqrtf(fmaxf(m[1] / p.D - rest * rest, 0.f) + p.eps);
        if (!live) continue;   // whole rows only: no barrier is skipped (TPR > 64 has one row per workgroup, live for all)
        if (lane == 0) {
            if (p.mean) p.mean[row] = mean;
            if (p.rstd) p.rstd[row] = rstd;
        }
        T* yr = static_cast<T*>(p.y) + row * p.ldy;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = (k * TPR + lane) * VW;
            if constexpr (KEEP)
                act8_store<VW>(v[k], c, p.Dp, p.codes + row * p.ldc, p.scales + row * p.lds);
            float o[VW];
#pragma unroll
            for (int i = 0; i < VW; ++i) o[i] = fmaf((v[k][i] - mean) * rstd, w[k][i], b[k][i]);
            store_cols(yr, c, p.D, o);
        }
    }
}

template <typename T, int TPR, int NV, bool KEPT>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void layer_norm_bwd_kernel(BwdParams p) {
    constexpr int BLOCK = TPR > 256 ? TPR : 256, ROWS = BLOCK / TPR, VW = RowType<T>::VW;
    __shared__ float red[2][2][16];
    const int lane = threadIdx.x % TPR, sub = threadIdx.x / TPR;
    float w[NV][VW], dw[NV][VW], db[NV][VW];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int c = (k * TPR + lane) * VW;
#pragma unroll
        for (int i = 0; i < VW; ++i) {
            w[k][i] = c + i < p.D ? (p.w ? p.w[c + i] : 1.f) : 0.f;
            dw[k][i] = db[k][i] = 0.f;
        }
    }
    int slot = 0;
    for (int64_t row0 = (int64_t)blockIdx.x * ROWS; row0 < p.M; row0 += (int64_t)gridDim.x * ROWS) {
        const bool live = row0 + sub < p.M;
        const int64_t row = live ? row0 + sub : p.M - 1;
        const T* gr = static_cast<const T*>(p.g) + row * p.ldg;
        const float mean = p.mean[row], rstd = p.rstd[row];
        float x[NV][VW], g[NV][VW], s[2] = {0.f, 0.f};
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = (k * TPR + lane) * VW;
            load_cols(gr, c, p.D, g[k]);
            if constexpr (KEPT)
                act8_load<VW>(p.codes + row * p.ldc, p.scales + row * p.lds, c, p.Dp, x[k]);
            else
                load_cols(static_cast<const T*>(p.x) + row * p.ldx, c, p.D, x[k]);
        }
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int i = 0; i < VW; ++i) {
                const float h = (x[k][i] - mean) * rstd, u = w[k][i] * g[k][i];
                s[0] += u;
                s[1] = fmaf(u, h, s[1]);
                if (live) {
                    dw[k][i] = fmaf(g[k][i], h, dw[k][i]);
                    db[k][i] += g[k][i];
                }
            }
        row_sum<TPR, 2>(s, red, slot);
        slot ^= 1;
        if (!live) continue;
        const float c0 = s[0] * p.inv_d, c1 = s[1] * p.inv_d;
        T* dr = static_cast<T*>(p.dx) + row * p.lddx;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = (k * TPR + lane) * VW;
            float o[VW];
#pragma unroll
            for (int i = 0; i < VW; ++i) {
                const float h = (x[k][i] - mean) * rstd;
                o[i] = rstd * (fmaf(w[k][i], g[k][i], -c0) - h * c1);
                if (p.leaky && !(x[k][i] > 0.f)) o[i] *= kLeakySlope;
            }
            store_cols(dr, c, p.D, o);
        }
    }
    // the workgroup's partial row of (dw, db): rows of a workgroup that share columns meet in LDS, in row order
    float* part = p.part + (int64_t)blockIdx.x * 2 * p.D;
    if constexpr (ROWS == 1) {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = (k * TPR + lane) * VW;
            store_cols(part, c, p.D, reinterpret_cast<const float(&)[4]>(dw[k][0]));
            store_cols(part + p.D, c, p.D, reinterpret_cast<const float(&)[4]>(db[k][0]));
            if constexpr (VW == 8) {
                store_cols(part, c + 4, p.D, reinterpret_cast<const float(&)[4]>(dw[k][4]));
                store_cols(part + p.D, c + 4, p.D, reinterpret_cast<const float(&)[4]>(db[k][4]));
            }
        }
    } else {
        __shared__ float join[ROWS > 1 ? BLOCK * VW : 1];   // one piece of every thread at a time: [sub][TPR * VW columns]
#pragma unroll
        for (int k = 0; k < NV; ++k) {
#pragma unroll
            for (int which = 0; which < 2; ++which) {
                __syncthreads();
#pragma unroll
                for (int i = 0; i < VW; ++i) join[threadIdx.x * VW + i] = which ? db[k][i] : dw[k][i];
                __syncthreads();
                for (int i = threadIdx.x; i < TPR * VW; i += BLOCK) {
                    const int c = k * TPR * VW + i;
                    float t = 0.f;
#pragma unroll
                    for (int r = 0; r < ROWS; ++r) t += join[r * TPR * VW + i];
                    if (c < p.D) part[which * p.D + c] = t;
                }
            }
        }
    }
}

// out[c] (+)= sum over the G partial rows: 64 columns per workgroup, 16 runs of rows side by side, joined in order
__global__ __launch_bounds__(1024) void column_join_kernel(const float* part, int G, int D, float* dw, float* db, int accumulate) {
    __shared__ float s[16][64];
    const int c = blockIdx.x * 64 + (threadIdx.x & 63), run = threadIdx.x >> 6;
    const int per = (G + 15) / 16, g0 = run * per, g1 = g0 + per < G ? g0 + per : G;
    float t = 0.f;
    if (c < 2 * D)
        for (int g = g0; g < g1; ++g) t += part[(int64_t)g * 2 * D + c];
    s[run][threadIdx.x & 63] = t;
    __syncthreads();
    if (run == 0 && c < 2 * D) {
#pragma unroll
        for (int r = 1; r < 16; ++r) t += s[r][threadIdx.x];
        float* out = c < D ? (dw ? dw + c : nullptr) : (db ? db + (c - D) : nullptr);
        if (out) *out = accumulate ? *out + t : t;
    }
}

// threads per row and 16-byte pieces per thread for a width: the fewest threads that cover the row with one piece each up to a wave,
// then up to 4 pieces per lane of a wave (no barrier), 256 threads, 1024 threads
struct Plan { int tpr, nv; };
Plan plan(int D, int vw) {
    const int pieces = (int)cdiv(D, vw);
    if (pieces <= 8) return {8, 1};
    if (pieces <= 16) return {16, 1};
    if (pieces <= 32) return {32, 1};
    if (pieces <= 64) return {64, 1};
    if (pieces <= 128) return {64, 2};
    if (pieces <= 256) return {64, 4};
    if (pieces <= 512) return {256, 2};
    if (pieces <= 1024) return {256, 4};
    if (pieces <= 2048) return {1024, 2};
    return {1024, 4};
}

template <typename F>
int with_plan(const Plan& pl, F f) {
#define PCVAE_LN_PLAN(t, n) if (pl.tpr == t && pl.nv == n) return f(std::integral_constant<int, t>{}, std::integral_constant<int, n>{})
    PCVAE_LN_PLAN(8, 1);
    PCVAE_LN_PLAN(16, 1);
    PCVAE_LN_PLAN(32, 1);
    PCVAE_LN_PLAN(64, 1);
    PCVAE_LN_PLAN(64, 2);
    PCVAE_LN_PLAN(64, 4);
    PCVAE_LN_PLAN(256, 2);
    PCVAE_LN_PLAN(256, 4);
    PCVAE_LN_PLAN(1024, 2);
    PCVAE_LN_PLAN(1024, 4);
#undef PCVAE_LN_PLAN
    set_error("layer_norm: no plan");
    return PCVAE_EINVAL;
}
template <typename F>
int with_type(int t, F f) {
    if (t == PCVAE_ROW_F32) return f((float*)nullptr);
    if (t == PCVAE_ROW_BF16) return f((__bf16*)nullptr);
    return f((_Float16*)nullptr);
}

int vector_width(int t) { return t == PCVAE_ROW_F32 ? 4 : 8; }
int rows_per_group(const Plan& pl) { return pl.tpr >= 256 ? 1 : 256 / pl.tpr; }
int bwd_groups(int64_t M, const Plan& pl) {
    const int64_t n = cdiv(M, rows_per_group(pl));
    return (int)(n < kBwdGroups ? n : kBwdGroups);
}

int check_rows(const char* who, int type, int64_t M, int D, int64_t ld, const void* p) {
    PCVAE_REQUIRE(row_type_ok(type), "%s: type %d is none of PCVAE_ROW_F32, PCVAE_ROW_BF16, PCVAE_ROW_F16", who, type);
    PCVAE_REQUIRE(M >= 0 && D >= 1 && D <= kMaxWidth, "%s: rows >= 0 and width in [1, %d] (got %lld x %d)", who, kMaxWidth, (long long)M, D);
    PCVAE_REQUIRE(M <= (1LL << 40), "%s: too many rows", who);
    PCVAE_REQUIRE(M == 0 || p, "%s: null rows", who);
    PCVAE_REQUIRE(M <= 1 || ld >= D, "%s: row stride %lld below the width %d", who, (long long)ld, D);
    return PCVAE_OK;
}

}  // namespace

extern "C" int pcvae_layer_norm_fwd(const void* x, int64_t ldx, int type, int64_t M, int D, const float* weight, const float* bias,
                                    float eps, void* y, int64_t ldy, float* mean, float* rstd, uint8_t* codes, int64_t ldc,
                                    uint8_t* scales, int64_t lds, pcvae_stream_t stream) {
    if (int rc = check_rows("layer_norm_fwd (x)", type, M, D, ldx, x)) return rc;
    if (int rc = check_rows("layer_norm_fwd (y)", type, M, D, ldy, y)) return rc;
    PCVAE_REQUIRE(eps >= 0.f, "layer_norm_fwd: eps %g is negative", (double)eps);
    PCVAE_REQUIRE((codes == nullptr) == (scales == nullptr), "layer_norm_fwd: codes and scales come together");
    if (codes) {
        if (int rc = act8_check("layer_norm", codes, ldc, scales, lds, M, D)) return rc;
    }
    if (M == 0) return PCVAE_OK;
    const Plan pl = plan(D, vector_width(type));
    FwdParams p{x, ldx, weight, bias, y, ldy, mean, rstd, codes, ldc, scales, lds, M, D, (int)cdiv(D, kAct8Block) * kAct8Block, eps};
    const int64_t groups = cdiv(M, rows_per_group(pl));
    const unsigned grid = (unsigned)(groups < 2048 ? groups : 2048);
    return with_type(type, [&](auto* tag) {
        using T = std::remove_pointer_t<decltype(tag)>;
        return with_plan(pl, [&](auto t, auto n) {
            constexpr int TPR = decltype(t)::value, NV = decltype(n)::value;
            const dim3 block(TPR > 256 ? TPR : 256);
            if (codes)
                hipLaunchKernelGGL((layer_norm_fwd_kernel<T, TPR, NV, true>), dim3(grid), block, 0, as_stream(stream), p);
            else
                hipLaunchKernelGGL((layer_norm_fwd_kernel<T, TPR, NV, false>), dim3(grid), block, 0, as_stream(stream), p);
            return check_launch("layer_norm_fwd");
        });
    });
}

extern "C" size_t pcvae_layer_norm_bwd_ws_bytes(int64_t M, int D, int type) {
    if (M <= 0 || D < 1 || D > kMaxWidth || !row_type_ok(type)) return 0;
    return (size_t)bwd_groups(M, plan(D, vector_width(type))) * 2 * D * sizeof(float);
}

extern "C" int pcvae_layer_norm_bwd(const void* g, int64_t ldg, int type, int64_t M, int D, const void* x, int64_t ldx,
                                    const uint8_t* codes, int64_t ldc, const uint8_t* scales, int64_t lds, const float* weight,
                                    const float* mean, const float* rstd, int leaky, void* dx, int64_t lddx, float* dweight,
                                    float* dbias, int accumulate, void* ws, size_t ws_bytes, pcvae_stream_t stream) {
    if (int rc = check_rows("layer_norm_bwd (g)", type, M, D, ldg, g)) return rc;
    if (int rc = check_rows("layer_norm_bwd (dx)", type, M, D, lddx, dx)) return rc;
    PCVAE_REQUIRE((x == nullptr) != (codes == nullptr) || M == 0, "layer_norm_bwd: the rows are either x or codes + scales");
    if (codes) {
        if (int rc = act8_check("layer_norm", codes, ldc, scales, lds, M, D)) return rc;
    } else {
        if (int rc = check_rows("layer_norm_bwd (x)", type, M, D, ldx, x)) return rc;
    }
    PCVAE_REQUIRE(M == 0 || (mean && rstd), "layer_norm_bwd: mean and rstd of the forward are needed");
    if (M == 0) {
        if (accumulate) return PCVAE_OK;
        if (dweight)
            if (int rc = pcvae_zero(dweight, (size_t)D * sizeof(float), stream)) return rc;
        if (dbias)
            if (int rc = pcvae_zero(dbias, (size_t)D * sizeof(float), stream)) return rc;
        return PCVAE_OK;
    }
    const size_t need = pcvae_layer_norm_bwd_ws_bytes(M, D, type);
    if (!ws || ws_bytes < need) {
        set_error("layer_norm_bwd: workspace too small (pcvae_layer_norm_bwd_ws_bytes)");
        return PCVAE_EWORKSPACE;
    }
    const Plan pl = plan(D, vector_width(type));
    const int G = bwd_groups(M, pl);
    BwdParams p{g, ldg, x, ldx, codes, ldc, scales, lds, weight, mean, rstd, dx, lddx, static_cast<float*>(ws), M, D,
                (int)cdiv(D, kAct8Block) * kAct8Block, leaky, 1.f / D};
    const int rc = with_type(type, [&](auto* tag) {
        using T = std::remove_pointer_t<decltype(tag)>;
        return with_plan(pl, [&](auto t, auto n) {
            constexpr int TPR = decltype(t)::value, NV = decltype(n)::value;
            const dim3 block(TPR > 256 ? TPR : 256);
            if (codes)
                hipLaunchKernelGGL((layer_norm_bwd_kernel<T, TPR, NV, true>), dim3(G), block, 0, as_stream(stream), p);
            else
                hipLaunchKernelGGL((layer_norm_bwd_kernel<T, TPR, NV, false>), dim3(G), block, 0, as_stream(stream), p);
            return check_launch("layer_norm_bwd");
        });
    });
    if (rc != PCVAE_OK || (!dweight && !dbias)) return rc;
    hipLaunchKernelGGL(column_join_kernel, dim3((unsigned)cdiv(2 * D, 64)), dim3(1024), 0, as_stream(stream), p.part, G, D, dweight, dbias,
                       accumulate);
    return check_launch("layer_norm_bwd (column sums)");
}
