// Activation checkpoints in 8 bits (act8.h) and their use in the backward pass of a linear layer:
//   pack     x [M, D] -> codes [M, 32 ceil(D / 32)] e4m3 + one scale byte per 32 columns          (1.03 bytes per value kept)
//   unpack   codes -> the values they stand for
//   leaky    g *= LeakyReLU'(x), read off the codes
//   weight   dW[N, K] = sum_m g[m, n] q[m, k],  db[n] = sum_m g[m, n]   from the codes of q [M, K]; with q behind a layer norm
//            (h = (q - mu_m) r_m, the layer's input w_k h + b_k):  dW = w_k (sum_m (g r_m) q - sum_m g r_m mu_m) + b_k db
#include "act8.h"

using namespace pcvae;

namespace {

// ---- pack / unpack / leaky: one lane per 16 bytes of x --------------------------------------------------------------------------
struct RowsParams {
    const void* x; int64_t ldx;
    void* y; int64_t ldy;
    uint8_t* codes; int64_t ldc; uint8_t* scales; int64_t lds;
    int64_t M; int D, Dp;
    unsigned pieces;   // lanes a row takes: Dp / VW
};

enum { ROWS_PACK = 0, ROWS_UNPACK = 1, ROWS_LEAKY = 2 };

template <typename T, int WHAT>
__global__ __launch_bounds__(256) void act8_rows_kernel(RowsParams p) {
    constexpr int VW = RowType<T>::VW;
    const int64_t total = p.M * p.pieces;   // a block's lanes (8 or 4) are neighbours: pieces is a multiple of them
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / p.pieces;
        const int c = (int)(i - row * p.pieces) * VW;
        float v[VW];
        if constexpr (WHAT == ROWS_PACK) {
            load_cols(static_cast<const T*>(p.x) + row * p.ldx, c, p.D, v);
            act8_store<VW>(v, c, p.Dp, p.codes + row * p.ldc, p.scales + row * p.lds);
        } else {
            act8_load<VW>(p.codes + row * p.ldc, p.scales + row * p.lds, c, p.Dp, v);
            T* y = static_cast<T*>(p.y) + row * p.ldy;
            if constexpr (WHAT == ROWS_LEAKY) {
                float g[VW];
                load_cols(y, c, p.D, g);
#pragma unroll
                for (int k = 0; k < VW; ++k) v[k] = v[k] > 0.f ? g[k] : kLeakySlope * g[k];
            }
            store_cols(y, c, p.D, v);
        }
    }
}

template <int WHAT>
int launch_rows(const char* what, int type, const RowsParams& p0, pcvae_stream_t stream) {
    RowsParams p = p0;
    if (p.M == 0) return PCVAE_OK;
    p.Dp = (int)cdiv(p.D, kAct8Block) * kAct8Block;
    p.pieces = p.Dp / (type == PCVAE_ROW_F32 ? 4 : 8);
    const int64_t groups = cdiv(p.M * p.pieces, 256);
    const dim3 grid((unsigned)(groups < 8192 ? groups : 8192));
    if (type == PCVAE_ROW_F32)
        hipLaunchKernelGGL((act8_rows_kernel<float, WHAT>), grid, dim3(256), 0, as_stream(stream), p);
    else if (type == PCVAE_ROW_BF16)
        hipLaunchKernelGGL((act8_rows_kernel<__bf16, WHAT>), grid, dim3(256), 0, as_stream(stream), p);
    else
        hipLaunchKernelGGL((act8_rows_kernel<_Float16, WHAT>), grid, dim3(256), 0, as_stream(stream), p);
    return check_launch(what);
}

int check_plain_rows(const char* who, int type, int64_t M, int64_t D, int64_t ld, const void* p) {
    PCVAE_REQUIRE(row_type_ok(type), "%s: type %d is none of PCVAE_ROW_F32, PCVAE_ROW_BF16, PCVAE_ROW_F16", who, type);
    PCVAE_REQUIRE(M == 0 || p, "%s: null rows", who);
    PCVAE_REQUIRE(M <= 1 || ld >= D, "%s: row stride %lld below the width %lld", who, (long long)ld, (long long)D);
    return PCVAE_OK;
}

// ---- weight gradient ------------------------------------------------------------------------------------------------------------
// A product's codes are exact in bf16 (act8.h), so fp32 g needs only its own split: g = c0 + c1 + c2 (three RNE bf16 components whose
// sum IS the fp32 value), three v_mfma_f32_32x32x16_bf16 per product, fp32 accumulate: fp32 products at a third of the bf16 rate.
// fp16 g is exact in two components, bf16 g in one; behind a norm the factor g r_m is an fp32 number again (three).
//
// One workgroup: 128 (n) x 128 (k) of dW over a range of rows m, four waves of 64 x 64.  Both operands run ALONG the contraction in
// memory's slow direction, so a chunk of 32 rows is turned on its way to LDS: a wave takes 8 consecutive rows, a lane holds the same
// column of all 8 - which is the 16-byte operand piece of an MFMA.  LDS image of an operand: [4 pieces of 8 rows][128 columns][16 bytes]
// (consecutive lanes, consecutive 16 bytes: no conflicts on either side).  Two stages, one barrier per chunk; the next chunk's loads are
// in flight over the products.
constexpr int TN = 128, TK = 128, TM = 32;
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));

struct DwParams {
    const void* g; int64_t ldg;
    const uint8_t* codes; int64_t ldc; const uint8_t* scales; int64_t lds;
    const float* mean; const float* rstd; const float* w; const float* b;   // the norm's, or null
    int64_t M; int N, K, Kp;
    int nn, nk, nz;            // tiles along n and k, ranges of m
    int64_t m_per;             // rows of a range, a multiple of TM
    float* part;               // [nz][nn nk][TN][TK] partial tiles (nz > 1), then [nz][nn TN] partial column sums
    float* part_db;
    float* dW; int64_t lddw; float* db; int accumulate;
};

// two fp32 values -> a word of two bf16 roundings, and back exactly
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    const bf16x2_t h = __builtin_convertvector((f32x2_t{a, b}), bf16x2_t);
    return __builtin_bit_cast(uint32_t, h);
}
__device__ __forceinline__ float low2(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float high2(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

template <int NC>
__device__ __forceinline__ void split8(const float (&v)[8], uint4 (&c)[NC]) {
    float r[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = v[i];
#pragma unroll
    for (int k = 0; k < NC; ++k) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            w[i] = pack2(r[2 * i], r[2 * i + 1]);
            if (k + 1 < NC) {
                r[2 * i] -= low2(w[i]);
                r[2 * i + 1] -= high2(w[i]);
            }
        }
        c[k] = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

template <typename T, int NC, bool NORM>
__global__ __launch_bounds__(256, 2) void act8_weight_kernel(DwParams p) {
    __shared__ uint4 sA[2][NC][4][TN];
    __shared__ uint4 sB[2][4][TK];
    float (*sSum)[4][TN] = reinterpret_cast<float (*)[4][TN]>(&sA[0][0][0][0]);   // column sums, behind the last product
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // logical order: all tiles of a range of rows next to each other (they share g and the codes in one XCD's L2)
    const int id = xcd_remap(blockIdx.x, gridDim.x);
    const int tiles = p.nn * p.nk, z = id / tiles, tile = id % tiles, tn = tile / p.nk, tk = tile % p.nk;
    const int64_t m0 = (int64_t)z * p.m_per, m1 = m0 + p.m_per < p.M ? m0 + p.m_per : p.M;
    const int chunks = (int)((m1 - m0 + TM - 1) / TM);

    // columns past the end read the last one: their products land in rows / columns of dW that are never stored
    const int na = min(tn * TN + lane, p.N - 1), nb = min(tn * TN + 64 + lane, p.N - 1);
    const int kc = min(tk * TK + 2 * lane, p.Kp - 2);
    const uint32_t sshift = 8 * ((kc >> 5) & 3);
    const T* g = static_cast<const T*>(p.g);
    const bool sums = NORM || (tk == 0 && p.db != nullptr);

    float ga[8], gb[8], mr[NORM ? 8 : 1];
    uint32_t q[8], sc[8];
    float suma = 0.f, sumb = 0.f, muca = 0.f, mucb = 0.f;

    auto fetch = [&](int chunk) {
        const int64_t base = m0 + (int64_t)chunk * TM + 8 * wave;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int64_t m = base + j < m1 ? base + j : m1 - 1;
            const T* gr = g + m * p.ldg;
            ga[j] = RowType<T>::one(gr + na);
            gb[j] = RowType<T>::one(gr + nb);
            q[j] = *reinterpret_cast<const uint16_t*>(p.codes + m * p.ldc + kc);
            sc[j] = *reinterpret_cast<const uint32_t*>(p.scales + m * p.lds + 4 * tk);
            if constexpr (NORM) {
                mr[j] = p.rstd[m];
            }
        }
    };
    auto place = [&](int chunk, int stage) {
        const int64_t base = m0 + (int64_t)chunk * TM + 8 * wave;
        if (base + 8 > m1) {   // rows from the range's end on count nothing
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (base + j >= m1) ga[j] = gb[j] = 0.f;
        }
        if (sums) {
            float s0 = 0.f, s1 = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) s0 += ga[j], s1 += gb[j];
            suma += s0;
            sumb += s1;
        }
        if constexpr (NORM) {
            float s0 = 0.f, s1 = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int64_t m = base + j < m1 ? base + j : m1 - 1;
                const float mu = p.mean[m];
                ga[j] *= mr[j];
                gb[j] *= mr[j];
                s0 = fmaf(ga[j], mu, s0);
                s1 = fmaf(gb[j], mu, s1);
            }
            muca += s0;
            mucb += s1;
        }
        uint4 ca[NC], cb[NC];
        split8<NC>(ga, ca);
        split8<NC>(gb, cb);
#pragma unroll
        for (int k = 0; k < NC; ++k) {
            sA[stage][k][wave][lane] = ca[k];
            sA[stage][k][wave][64 + lane] = cb[k];
        }
        uint32_t lo[4], hi[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t e[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float s = act8_scale((sc[2 * j + i] >> sshift) & 0xffu);
                e[i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q[2 * j + i], s, false));
            }
            lo[j] = __builtin_amdgcn_perm(e[1], e[0], 0x05040100u);
            hi[j] = __builtin_amdgcn_perm(e[1], e[0], 0x07060302u);
        }
        sB[stage][wave][2 * lane] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        sB[stage][wave][2 * lane + 1] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    };

    const int wn = (wave >> 1) * 64, wk = (wave & 1) * 64;
    f32x16_t acc[2][2];
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[a][b][i] = 0.f;

    fetch(0);
    place(0, 0);
    if (chunks > 1) fetch(1);
    __syncthreads();
    for (int c = 0; c < chunks; ++c) {
        const int stage = c & 1;
        if (c + 1 < chunks) place(c + 1, stage ^ 1);
        if (c + 2 < chunks) fetch(c + 2);
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int piece = 2 * s + (lane >> 5), l = lane & 31;
            bf16x8_t b[2];
#pragma unroll
            for (int t = 0; t < 2; ++t) b[t] = __builtin_bit_cast(bf16x8_t, sB[stage][piece][wk + 32 * t + l]);
#pragma unroll
            for (int k = NC - 1; k >= 0; --k)   // the smallest components first
#pragma unroll
                for (int a = 0; a < 2; ++a) {
                    const bf16x8_t av = __builtin_bit_cast(bf16x8_t, sA[stage][k][piece][wn + 32 * a + l]);
#pragma unroll
                    for (int t = 0; t < 2; ++t) acc[a][t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(av, b[t], acc[a][t], 0, 0, 0);
                }
        }
        __syncthreads();
    }

    if (sums) {
        sSum[0][wave][lane] = suma;
        sSum[0][wave][64 + lane] = sumb;
        if constexpr (NORM) {
            sSum[1][wave][lane] = muca;
            sSum[1][wave][64 + lane] = mucb;
        }
        __syncthreads();
    }
    auto total = [&](int which, int n) { return (sSum[which][0][n] + sSum[which][1][n]) + (sSum[which][2][n] + sSum[which][3][n]); };
    if (tk == 0 && p.db != nullptr && threadIdx.x < TN) {
        const int n = tn * TN + threadIdx.x;
        const float t = total(0, threadIdx.x);
        if (p.nz > 1) p.part_db[(int64_t)z * p.nn * TN + n] = t;
        else if (n < p.N) p.db[n] = p.accumulate ? p.db[n] + t : t;
    }
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int kk = wk + 32 * t + (lane & 31), k = tk * TK + kk;
            const bool inside = k < p.K;
            float wv = 1.f, bv = 0.f;
            if constexpr (NORM) {
                wv = p.w && inside ? p.w[k] : 1.f;
                bv = p.b && inside ? p.b[k] : 0.f;
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int nr = wn + 32 * a + (i & 3) + 8 * (i >> 2) + 4 * (lane >> 5), n = tn * TN + nr;
                float v = acc[a][t][i];
                if constexpr (NORM) v -= total(1, nr);
                if constexpr (NORM) v = fmaf(wv, v, bv * total(0, nr));
                if (p.nz > 1) {
                    p.part[(((int64_t)z * tiles + tile) * TN + nr) * TK + kk] = v;
                } else if (inside && n < p.N) {
                    float* out = p.dW + (int64_t)n * p.lddw + k;
                    *out = p.accumulate ? *out + v : v;
                }
            }
        }
}

// the ranges of rows joined in order
__global__ __launch_bounds__(256) void act8_weight_join_kernel(DwParams p) {
    const int tiles = p.nn * p.nk;
    const int64_t total = (int64_t)tiles * TN * TK / 4;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int tile = (int)(i / (TN * TK / 4)), e = (int)(i % (TN * TK / 4)) * 4;
        const int n = tile / p.nk * TN + e / TK, k = tile % p.nk * TK + e % TK;
        if (n >= p.N || k >= p.K) continue;
        f32x4_t s = {0.f, 0.f, 0.f, 0.f};
        for (int z = 0; z < p.nz; ++z)
            s += *reinterpret_cast<const f32x4_t*>(p.part + ((int64_t)z * tiles + tile) * TN * TK + e);
        float* out = p.dW + (int64_t)n * p.lddw + k;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (k + j < p.K) out[j] = p.accumulate ? out[j] + s[j] : s[j];
    }
    if (p.db) {
        for (int64_t n = (int64_t)blockIdx.x * 256 + threadIdx.x; n < p.N; n += (int64_t)gridDim.x * 256) {
            float s = 0.f;
            for (int z = 0; z < p.nz; ++z) s += p.part_db[(int64_t)z * p.nn * TN + n];
            p.db[n] = p.accumulate ? p.db[n] + s : s;
        }
    }
}

__global__ __launch_bounds__(256) void act8_weight_empty_kernel(DwParams p) {
    const int64_t total = (int64_t)p.N * p.K;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        p.dW[i / p.K * p.lddw + i % p.K] = 0.f;
        if (p.db && i < p.N) p.db[i] = 0.f;
    }
}

// ranges of rows: enough workgroups for two per CU, each at least 8 chunks long (a shorter range costs more in its partial tile than
// it gives)
struct DwPlan { int nn, nk, nz; int64_t m_per; };
DwPlan dw_plan(int64_t M, int64_t N, int64_t K) {
    DwPlan d;
    d.nn = (int)cdiv(N, TN);
    d.nk = (int)cdiv(K, TK);
    const int64_t tiles = (int64_t)d.nn * d.nk;
    int64_t nz = tiles >= 512 ? 1 : 512 / tiles;
    const int64_t most = cdiv(M, 8 * TM);
    if (nz > most) nz = most;
    if (nz < 1) nz = 1;
    d.m_per = cdiv(cdiv(M, nz), TM) * TM;
    d.nz = (int)cdiv(M, d.m_per);
    return d;
}
size_t dw_ws(const DwPlan& d) {
    return d.nz > 1 ? ((size_t)d.nz * d.nn * d.nk * TN * TK + (size_t)d.nz * d.nn * TN) * sizeof(float) : 0;
}

template <typename T, int NC>
int launch_dw(const DwParams& p, pcvae_stream_t stream) {
    const dim3 grid((unsigned)(p.nn * p.nk * p.nz));
    if (p.mean)
        hipLaunchKernelGGL((act8_weight_kernel<T, 3, true>), grid, dim3(256), 0, as_stream(stream), p);
    else
        hipLaunchKernelGGL((act8_weight_kernel<T, NC, false>), grid, dim3(256), 0, as_stream(stream), p);
    if (int rc = check_launch("act8_bwd_weight")) return rc;
    if (p.nz == 1) return PCVAE_OK;
    const int64_t groups = cdiv((int64_t)p.nn * p.nk * TN * TK / 4, 256);
    hipLaunchKernelGGL(act8_weight_join_kernel, dim3((unsigned)(groups < 4096 ? groups : 4096)), dim3(256), 0, as_stream(stream), p);
    return check_launch("act8_bwd_weight (join)");
}

}  // namespace

extern "C" int pcvae_act8_pack(const void* x, int64_t ldx, int type, int64_t M, int64_t D, uint8_t* codes, int64_t ldc, uint8_t* scales,
                               int64_t lds, pcvae_stream_t stream) {
    if (int rc = act8_check("act8_pack", codes, ldc, scales, lds, M, D)) return rc;
    if (int rc = check_plain_rows("act8_pack", type, M, D, ldx, x)) return rc;
    RowsParams p{x, ldx, nullptr, 0, codes, ldc, scales, lds, M, (int)D, 0, 0};
    return launch_rows<ROWS_PACK>("act8_pack", type, p, stream);
}

extern "C" int pcvae_act8_unpack(const uint8_t* codes, int64_t ldc, const uint8_t* scales, int64_t lds, int64_t M, int64_t D, void* y,
                                 int64_t ldy, int type, pcvae_stream_t stream) {
    if (int rc = act8_check("act8_unpack", codes, ldc, scales, lds, M, D)) return rc;
    if (int rc = check_plain_rows("act8_unpack", type, M, D, ldy, y)) return rc;
    RowsParams p{nullptr, 0, y, ldy, const_cast<uint8_t*>(codes), ldc, const_cast<uint8_t*>(scales), lds, M, (int)D, 0, 0};
    return launch_rows<ROWS_UNPACK>("act8_unpack", type, p, stream);
}

extern "C" int pcvae_act8_leaky_bwd(void* g, int64_t ldg, int type, const uint8_t* codes, int64_t ldc, const uint8_t* scales, int64_t lds,
                                    int64_t M, int64_t D, pcvae_stream_t stream) {
    if (int rc = act8_check("act8_leaky_bwd", codes, ldc, scales, lds, M, D)) return rc;
    if (int rc = check_plain_rows("act8_leaky_bwd", type, M, D, ldg, g)) return rc;
    RowsParams p{nullptr, 0, g, ldg, const_cast<uint8_t*>(codes), ldc, const_cast<uint8_t*>(scales), lds, M, (int)D, 0, 0};
    return launch_rows<ROWS_LEAKY>("act8_leaky_bwd", type, p, stream);
}

extern "C" size_t pcvae_act8_bwd_weight_ws_bytes(int64_t M, int64_t N, int64_t K) {
    if (M <= 0 || N <= 0 || K <= 0) return 0;
    return dw_ws(dw_plan(M, N, K));
}

extern "C" int pcvae_act8_bwd_weight(const void* g, int64_t ldg, int type, const uint8_t* codes, int64_t ldc, const uint8_t* scales,
                                     int64_t lds, int64_t M, int64_t N, int64_t K, const float* mean, const float* rstd,
                                     const float* weight, const float* bias, float* dW, int64_t lddw, float* db, int accumulate, void* ws,
                                     size_t ws_bytes, pcvae_stream_t stream) {
    if (int rc = act8_check("act8_bwd_weight", codes, ldc, scales, lds, M, K)) return rc;
    if (int rc = check_plain_rows("act8_bwd_weight", type, M, N, ldg, g)) return rc;
    PCVAE_REQUIRE(N >= 1 && N <= (1 << 24) && dW, "act8_bwd_weight: dW [N, K], N in [1, 2^24]");
    PCVAE_REQUIRE(N == 1 || lddw >= K, "act8_bwd_weight: row stride %lld of dW below its width %lld", (long long)lddw, (long long)K);
    PCVAE_REQUIRE((mean == nullptr) == (rstd == nullptr), "act8_bwd_weight: mean and rstd come together");
    PCVAE_REQUIRE(mean || (!weight && !bias), "act8_bwd_weight: the norm's weight / bias need its mean and rstd");
    DwParams p{g, ldg, codes, ldc, scales, lds, mean, rstd, weight, bias, M, (int)N, (int)K, (int)cdiv(K, kAct8Block) * kAct8Block,
               0, 0, 0, 0, nullptr, nullptr, dW, lddw, db, accumulate};
    if (M == 0) {
        if (accumulate) return PCVAE_OK;
        const int64_t groups = cdiv(N * K, 256);
        hipLaunchKernelGGL(act8_weight_empty_kernel, dim3((unsigned)(groups < 4096 ? groups : 4096)), dim3(256), 0, as_stream(stream), p);
        return check_launch("act8_bwd_weight");
    }
    const DwPlan d = dw_plan(M, N, K);
    PCVAE_REQUIRE((int64_t)d.nn * d.nk * d.nz < (1LL << 31), "act8_bwd_weight: launch too large");
    const size_t need = dw_ws(d);
    if (need && (!ws || ws_bytes < need)) {
        set_error("act8_bwd_weight: workspace too small (pcvae_act8_bwd_weight_ws_bytes)");
        return PCVAE_EWORKSPACE;
    }
    p.nn = d.nn; p.nk = d.nk; p.nz = d.nz; p.m_per = d.m_per;
    p.part = static_cast<float*>(ws);
    p.part_db = need ? p.part + (size_t)d.nz * d.nn * d.nk * TN * TK : nullptr;
    if (type == PCVAE_ROW_F32) return launch_dw<float, 3>(p, stream);
    if (type == PCVAE_ROW_BF16) return launch_dw<__bf16, 1>(p, stream);
    return launch_dw<_Float16, 2>(p, stream);
}
