// Layer norm over the rows of x [M, D], forward and backward, with the reduction of the weight's and the bias's gradient.
//
//   mu = mean x,  r = 1 / sqrt(mean (x - mu)^2 + eps),  h = (x - mu) r,  y = w h + b
//   dx = r (w g - mean(w g) - h mean(w g h))  [* LeakyReLU'(x): x a LeakyReLU's output],   dw = sum_m g h,   db = sum_m g
//
// Both directions read every operand once and keep the row in registers between the passes over it (the variance is taken about the
// mean, not from a difference of moments; rows whose squares or sum leave fp32's range are taken at 2^-80 of their size, so every finite row
// has its statistics, and a row that holds NaN or an infinity has NaN for both); statistics and sums are fp32.  TPR neighbouring threads own a row, each holds NV pieces of
// 16 bytes of it (8 lanes to 16 waves; rule: plan()).  Any of the row types fp32 / bf16 / fp16, any width up to 16384, any row
// stride.  The forward optionally also writes the row's 8-bit form (act8.h), and the backward takes x from it: the norm's saved input
// is then one byte per value, and LeakyReLU' reads off its codes.
//
// The backward's column sums: a thread owns columns, so dw and db accumulate in its registers over all rows of its workgroup; the
// workgroups' partial rows [G, 2, D] are joined in workgroup order by a second kernel (no atomics: the same bits every run).
//
// Bound: memory.  Beside a device copy's rate (4.96 TB/s over 2 x 2 GiB): forward 32768 x 2048 bf16 56 us = 4.8 TB/s, 16384 x 2048 fp32
// keeping its 8-bit form 54 us = 5.6 TB/s (inputs partly cached); backward 32768 x 2048 bf16 83 us = 4.9 TB/s, 16384 x 2048 fp32 from its
// 8-bit form 52 us = 5.9 TB/s; one row of 256 1.8 us.  Past 8192 columns the backward does not fit its registers (plan()): 4096 x 16384
// fp32 229 us = 3.5 TB/s, bf16 99 us = 4.1 TB/s, from the 8-bit form 231 and 155 us; the forward holds 5.6 and 5.0 TB/s there.
// A piece is one 16-byte load whatever the width and alignment of the rows (value-by-value tails behind branches: 104 / 129 us instead
// of 56 / 82 on the bf16 case), and the next row's loads are in flight over the current row's sums.
#include "act8.h"

using namespace pcvae;

namespace {

constexpr int kMaxWidth = 16384;

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

// the next row's loads are issued before the current row's sums: they are in flight over two reductions and the stores
template <typename T, int TPR, int NV, int END, bool KEEP>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void layer_norm_fwd_kernel(FwdParams p) {
    constexpr int BLOCK = TPR > 256 ? TPR : 256, ROWS = BLOCK / TPR, VW = RowType<T>::VW;
    __shared__ float red0[2][1][16], red1[2][2][16];
    const int lane = threadIdx.x % TPR, sub = threadIdx.x / TPR;
    const int tail = p.D / VW / TPR;   // the piece index the row's end falls into (pieces behind it are empty)
    float w[NV][VW], b[NV][VW];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int c = (k * TPR + lane) * VW;
        param_load<VW>(p.w, c, p.D, END, k >= tail, 1.f, w[k]);
        param_load<VW>(p.b, c, p.D, END, k >= tail, 0.f, b[k]);
    }
    const T* x = static_cast<const T*>(p.x);
    const int64_t step = (int64_t)gridDim.x * ROWS;
    auto row_at = [&](int64_t row0) { return x + (row0 + sub < p.M ? row0 + sub : p.M - 1) * p.ldx; };
    Raw<16> next[NV];
    int64_t row0 = (int64_t)blockIdx.x * ROWS;
#pragma unroll
    for (int k = 0; k < NV; ++k) next[k] = piece_load<T>(row_at(row0), (k * TPR + lane) * VW, p.D, END);
    for (; row0 < p.M; row0 += step) {
        const bool live = row0 + sub < p.M;
        const int64_t row = live ? row0 + sub : p.M - 1;
        float v[NV][VW], s[1] = {0.f}, m[2] = {0.f, 0.f};
#pragma unroll
        for (int k = 0; k < NV; ++k) piece_values<T>(next[k], row_at(row0), (k * TPR + lane) * VW, p.D, END, k >= tail, v[k]);
        if (row0 + step < p.M) {
#pragma unroll
            for (int k = 0; k < NV; ++k) next[k] = piece_load<T>(row_at(row0 + step), (k * TPR + lane) * VW, p.D, END);
        }
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int i = 0; i < VW; ++i) s[0] += v[k][i];
        row_sum<TPR, 1>(s, red0, 0);
        const float near = s[0] / p.D;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = (k * TPR + lane) * VW;
#pragma unroll
            for (int i = 0; i < VW; ++i) {
                const float d = END == ROW_FULL || c + i < p.D ? v[k][i] - near : 0.f;
                m[0] += d;
                m[1] = fmaf(d, d, m[1]);
            }
        }
        // what the first sum's roundings left of the mean shows in the deviations' own mean: rows far from zero (and constant ones) need it
        row_sum<TPR, 2>(m, red1, 0);
        const float rest = m[0] / p.D;
        float mean = near + rest, rstd = 1.f / sqrtf(fmaxf(m[1] / p.D - rest * rest, 0.f) + p.eps);
        if (!(m[1] < INFINITY)) {   // (the same for every thread of a row; rows of more than a wave have their workgroup to themselves)
            // Squares or the sum out of fp32's range: the statistics again, of the row times 2^-80 - its values are then below 2^48, the sums
            // below 2^110, and what vanishes is under 2^-80 of the largest deviation.  A row that holds NaN or an infinity stays NaN.
            float far[1] = {0.f}, dev[2] = {0.f, 0.f};
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int i = 0; i < VW; ++i) far[0] = fmaf(v[k][i], 0x1p-80f, far[0]);
            row_sum<TPR, 1>(far, red0, 0);
            const float mid = far[0] / p.D;
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const int c = (k * TPR + lane) * VW;
#pragma unroll
                for (int i = 0; i < VW; ++i) {
                    const float d = END == ROW_FULL || c + i < p.D ? fmaf(v[k][i], 0x1p-80f, -mid) : 0.f;
                    dev[0] += d;
                    dev[1] = fmaf(d, d, dev[1]);
                }
            }
            row_sum<TPR, 2>(dev, red1, 0);
            const float left = dev[0] / p.D, var = dev[1] / p.D - left * left;
            const float sum = (var < 0.f ? 0.f : var) + p.eps * 0x1p-80f * 0x1p-80f;
            mean = (mid + left) * 0x1p80f;
            rstd = sum == 0.f ? 1.f / sqrtf(p.eps) : 0x1p-80f / sqrtf(sum);
        }
        if (!live) continue;   // whole rows only: no barrier is skipped (TPR > 64 has one row per workgroup, live for all)
        if (lane == 0) {
            if (p.mean) p.mean[row] = mean;
            if (p.rstd) p.rstd[row] = rstd;
        }
        T* yr = static_cast<T*>(p.y) + row * p.ldy;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = (k * TPR + lane) * VW;
            if constexpr (KEEP) act8_store<T>(v[k], c, p.Dp, p.codes + row * p.ldc, act8_scale_at(p.scales, p.lds, row, c));
            float o[VW];
#pragma unroll
            for (int i = 0; i < VW; ++i) o[i] = fmaf((v[k][i] - mean) * rstd, w[k][i], b[k][i]);
            piece_store<T>(yr, c, p.D, END, o);
        }
    }
}

template <typename T, int TPR, int NV, int END, bool KEPT>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void layer_norm_bwd_kernel(BwdParams p) {
    constexpr int BLOCK = TPR > 256 ? TPR : 256, ROWS = BLOCK / TPR, VW = RowType<T>::VW;
    __shared__ float red[2][2][16];
    const int lane = threadIdx.x % TPR, sub = threadIdx.x / TPR;
    const int tail = p.D / VW / TPR;
    float w[NV][VW], dw[NV][VW], db[NV][VW];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        param_load<VW>(p.w, (k * TPR + lane) * VW, p.D, END, k >= tail, 1.f, w[k]);
#pragma unroll
        for (int i = 0; i < VW; ++i) dw[k][i] = db[k][i] = 0.f;
    }
    const int64_t step = (int64_t)gridDim.x * ROWS;
    auto row_of = [&](int64_t row0) { return row0 + sub < p.M ? row0 + sub : p.M - 1; };
    struct Loaded {
        Raw<16> g[NV], x[KEPT ? 1 : NV];
        Raw<VW> q[KEPT ? NV : 1];
        uint32_t s[KEPT ? NV : 1];
        float mean, rstd;
    } next;
    auto load = [&](int64_t row0) {
        const int64_t row = row_of(row0);
        next.mean = p.mean[row];
        next.rstd = p.rstd[row];
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = (k * TPR + lane) * VW;
            next.g[k] = piece_load<T>(static_cast<const T*>(p.g) + row * p.ldg, c, p.D, END);
            if constexpr (KEPT) {
                const int cc = c < p.Dp ? c : p.Dp - VW;
                next.q[k] = *reinterpret_cast<const Raw<VW>*>(p.codes + row * p.ldc + cc);
                next.s[k] = *act8_scale_at(p.scales, p.lds, row, cc);
            } else {
                next.x[k] = piece_load<T>(static_cast<const T*>(p.x) + row * p.ldx, c, p.D, END);
            }
        }
    };
    int slot = 0;
    int64_t row0 = (int64_t)blockIdx.x * ROWS;
    load(row0);
    for (; row0 < p.M; row0 += step) {
        const bool live = row0 + sub < p.M;
        const int64_t row = row_of(row0);
        const float mean = next.mean, rstd = next.rstd;
        float x[NV][VW], g[NV][VW], s[2] = {0.f, 0.f};
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = (k * TPR + lane) * VW;
            piece_values<T>(next.g[k], static_cast<const T*>(p.g) + row * p.ldg, c, p.D, END, k >= tail, g[k]);
            if constexpr (KEPT) {
                const float scale = act8_scale(next.s[k]);   // columns behind the row read its last codes: their g and w are 0
                act8_values(next.q[k].w[0], scale, x[k]);
                if constexpr (VW == 8) act8_values(next.q[k].w[1], scale, x[k] + 4);
                if (END != ROW_FULL && c >= p.Dp) {
#pragma unroll
                    for (int i = 0; i < VW; ++i) x[k][i] = 0.f;
                }
            } else {
                piece_values<T>(next.x[k], static_cast<const T*>(p.x) + row * p.ldx, c, p.D, END, k >= tail, x[k]);
            }
        }
        if (row0 + step < p.M) load(row0 + step);
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
            piece_store<T>(dr, c, p.D, END, o);
        }
    }
    // the workgroup's partial row of (dw, db): rows of a workgroup that share columns meet in LDS, in row order
    float* part = p.part + (int64_t)blockIdx.x * 2 * p.D;
    if constexpr (ROWS == 1) {
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int h = 0; h < VW; h += 4) {
                const int c = (k * TPR + lane) * VW + h;
                const float a[4] = {dw[k][h], dw[k][h + 1], dw[k][h + 2], dw[k][h + 3]};
                const float e[4] = {db[k][h], db[k][h + 1], db[k][h + 2], db[k][h + 3]};
                piece_store<float>(part, c, p.D, END, a);
                piece_store<float>(part + p.D, c, p.D, END, e);
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

// out[c] (+)= sum over the G partial rows: 32 columns per workgroup, 32 runs of rows side by side (eight rows of a run in flight), the runs
// joined in order
__global__ __launch_bounds__(1024) void column_join_kernel(const float* part, int G, int D, float* dw, float* db, int accumulate) {
    __shared__ float s[32][33];
    const int col = threadIdx.x & 31, run = threadIdx.x >> 5, c = blockIdx.x * 32 + col;
    const int per = (G + 31) / 32, g0 = run * per, g1 = g0 + per < G ? g0 + per : G;
    float t = 0.f;
    if (c < 2 * D) {
        const float* q = part + c;
        for (int g = g0; g < g1; g += 8) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = g + i < g1 ? q[(int64_t)(g + i) * 2 * D] : 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) t += v[i];
        }
    }
    s[run][col] = t;
    __syncthreads();
    if (run == 0 && c < 2 * D) {
#pragma unroll
        for (int r = 1; r < 32; ++r) t += s[r][col];
        float* out = c < D ? (dw ? dw + c : nullptr) : (db ? db + (c - D) : nullptr);
        if (out) *out = accumulate ? *out + t : t;
    }
}

// threads per row and 16-byte pieces per thread for a width: one piece each up to a wave, then more pieces per lane of a wave (no barrier)
// as far as the registers of the backward go - it holds w, dw, db in fp32 per column: 4 pieces of fp32, 2 of the half types -, then 256
// threads, then 1024.  The last rung (8193 .. 16384 columns) has as many pieces in 1024 threads, where a thread has 128 registers: the
// backward spills 10 to 58 of them there (28 to 212 bytes of scratch per lane), the forward none.
struct Plan { int tpr, nv, end; };
Plan plan(int D, int vw) {
    const int pieces = (int)cdiv(D, vw);
    Plan pl{1024, vw == 4 ? 4 : 2, 0};
    const int few[4] = {8, 16, 32, 64};
    for (int t : few)
        if (pieces <= t) { pl = {t, 1, 0}; break; }
    if (pieces > 64) {
        if (pieces <= 128) pl = {64, 2, 0};
        else if (pieces <= 256 && vw == 4) pl = {64, 4, 0};
        else if (pieces <= 256) pl = {256, 1, 0};
        else if (pieces <= 512) pl = {256, 2, 0};
        else if (pieces <= 1024 && vw == 4) pl = {256, 4, 0};
        else if (pieces <= 1024) pl = {1024, 1, 0};
        else if (pieces <= 2048) pl = {1024, 2, 0};
    }
    pl.end = row_end(D, vw, pl.tpr * pl.nv * vw);
    return pl;
}

template <int VW, typename F>
int with_plan(const Plan& pl, F f) {
#define PCVAE_LN_PLAN(t, n)                                                                                                          \
    if (pl.tpr == t && pl.nv == n) {                                                                                                 \
        if (pl.end == ROW_FULL) return f(std::integral_constant<int, t>{}, std::integral_constant<int, n>{}, std::integral_constant<int, 0>{}); \
        return f(std::integral_constant<int, t>{}, std::integral_constant<int, n>{}, std::integral_constant<int, 1>{});              \
    }
    if (pl.end == ROW_TINY) return f(std::integral_constant<int, 8>{}, std::integral_constant<int, 1>{}, std::integral_constant<int, 2>{});
    PCVAE_LN_PLAN(8, 1)
    PCVAE_LN_PLAN(16, 1)
    PCVAE_LN_PLAN(32, 1)
    PCVAE_LN_PLAN(64, 1)
    PCVAE_LN_PLAN(64, 2)
    PCVAE_LN_PLAN(256, 2)
    PCVAE_LN_PLAN(1024, 2)
    if constexpr (VW == 4) {
        PCVAE_LN_PLAN(64, 4)
        PCVAE_LN_PLAN(256, 4)
        PCVAE_LN_PLAN(1024, 4)
    } else {
        PCVAE_LN_PLAN(256, 1)
        PCVAE_LN_PLAN(1024, 1)
    }
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
// Workgroups of a launch at most.  A forward's loads its parameters once per workgroup (1024 / 4096, measured on 8192 x 5397 fp32: 76 / 81 us
// with 1024 threads per row, on 32768 x 2048 bf16: 62 / 58 us with 256); each of a backward's leaves a partial row of column sums (256 / 512 /
// 768: 8192 x 5397 fp32 108 / 116 / 124 us, 32768 x 2048 bf16 118 / 84 / 83 us, 65536 x 256 fp32 from codes 60 / 40 / 36 us)
int fwd_groups(int64_t M, const Plan& pl) {
    const int64_t n = cdiv(M, rows_per_group(pl)), most = pl.tpr == 1024 ? 1024 : 4096;
    return (int)(n < most ? n : most);
}
int bwd_groups(int64_t M, const Plan& pl) {
    const int64_t n = cdiv(M, rows_per_group(pl)), most = pl.tpr == 1024 ? 256 : (pl.tpr <= 64 && pl.nv == 1 ? 768 : 512);
    return (int)(n < most ? n : most);
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
    const unsigned grid = (unsigned)fwd_groups(M, pl);
    return with_type(type, [&](auto* tag) {
        using T = std::remove_pointer_t<decltype(tag)>;
        return with_plan<RowType<T>::VW>(pl, [&](auto t, auto n, auto e) {
            constexpr int TPR = decltype(t)::value, NV = decltype(n)::value, END = decltype(e)::value;
            const dim3 block(TPR > 256 ? TPR : 256);
            if (codes)
                hipLaunchKernelGGL((layer_norm_fwd_kernel<T, TPR, NV, END, true>), dim3(grid), block, 0, as_stream(stream), p);
            else
                hipLaunchKernelGGL((layer_norm_fwd_kernel<T, TPR, NV, END, false>), dim3(grid), block, 0, as_stream(stream), p);
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
        return with_plan<RowType<T>::VW>(pl, [&](auto t, auto n, auto e) {
            constexpr int TPR = decltype(t)::value, NV = decltype(n)::value, END = decltype(e)::value;
            const dim3 block(TPR > 256 ? TPR : 256);
            if (codes)
                hipLaunchKernelGGL((layer_norm_bwd_kernel<T, TPR, NV, END, true>), dim3(G), block, 0, as_stream(stream), p);
            else
                hipLaunchKernelGGL((layer_norm_bwd_kernel<T, TPR, NV, END, false>), dim3(G), block, 0, as_stream(stream), p);
            return check_launch("layer_norm_bwd");
        });
    });
    if (rc != PCVAE_OK || (!dweight && !dbias)) return rc;
    hipLaunchKernelGGL(column_join_kernel, dim3((unsigned)cdiv(2 * D, 32)), dim3(1024), 0, as_stream(stream), p.part, G, D, dweight, dbias,
                       accumulate);
    return check_launch("layer_norm_bwd (column sums)");
}
