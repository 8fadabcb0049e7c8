// Activation checkpoints in 8 bits (act8.h) and their use in the backward pass of a linear layer:
//   pack     x [M, D] -> codes [M, 32 ceil(D / 32)] e4m3 + one scale byte per 32 columns          (1.03 bytes per value kept)
//   unpack   codes -> the values they stand for
//   leaky    g *= LeakyReLU'(x), read off the codes
//   weight   dW[N, K] = sum_m g[m, n] q[m, k],  db[n] = sum_m g[m, n]   from the codes of q [M, K]; with q behind a layer norm
//            (h = (q - mu_m) r_m, the layer's input w_k h + b_k):  dW = w_k (sum_m (g r_m) q - sum_m g r_m mu_m) + b_k db
//
// Bounds.  The row kernels: memory (8192 x 5397 fp32 pack 53 us = 4.2 TB/s of codes and values, unpack 35 us, the codes partly cached;
// LeakyReLU' over 8192 x 256 fp32 7 us, over 32768 x 2048 fp32 102 us; a device copy runs at 4.96 TB/s).  The weight gradient: the matrix pipe -
// 4864 x 1024 over 32768 rows, fp32 g, 923 us (868 at best) = 354 TFLOP/s of fp32-exact products = 1061 TFLOP/s of bf16 products issued, 0.87
// of what the library's largest bf16 product reaches (1222); its pipe is 0.52 busy by the counters, 8 registers spill - and, for one
// component (bf16 g), the instructions around its products: 2048 x 2048 over 16384 rows 178 us = 773 TFLOP/s (matrix pipe 0.35 busy, LDS 0.26, vector
// issue 0.27: two waves per SIMD do not cover each other's waits); two components (fp16 g) 257 us, behind a norm three whatever g's type: 340-370
// us.  Small ones are launches and latency: 256 x 256 over 8192 rows 24 us.
#include "act8.h"

using namespace pcvae;

namespace {

// ---- pack / unpack / leaky: one lane per 16 bytes of x --------------------------------------------------------------------------
struct RowsParams {
    const void* x; int64_t ldx;
    void* y; int64_t ldy;
    uint8_t* codes; int64_t ldc; uint8_t* scales; int64_t lds;
    int64_t M; int D, Dp;
    int pieces, end;              // lanes a row takes: Dp / VW;  RowEnd
    int64_t step_rows; int step;  // the launch's lanes = step_rows rows + step pieces
};

enum { ROWS_PACK = 0, ROWS_UNPACK = 1, ROWS_LEAKY = 2 };

// Lanes run along the rows back to back (a block's 8 or 4 lanes are neighbours: pieces is a multiple of them); a thread walks the launch's
// stride in (row, piece) steps - one division per thread -, the next piece's loads in flight over the current one.
template <typename T, int WHAT>
__global__ __launch_bounds__(256) void act8_rows_kernel(RowsParams p) {
    constexpr int VW = RowType<T>::VW;
    const int64_t first = (int64_t)blockIdx.x * 256 + threadIdx.x;
    int64_t row = first / p.pieces;
    int piece = (int)(first - row * p.pieces);
    Raw<16> x{};
    Raw<VW> q{};
    uint32_t byte = 0;
    auto load = [&](int64_t row, int c) {
        if constexpr (WHAT == ROWS_PACK) x = piece_load<T>(static_cast<const T*>(p.x) + row * p.ldx, c, p.D, p.end);
        if constexpr (WHAT == ROWS_LEAKY) x = piece_load<T>(static_cast<const T*>(p.y) + row * p.ldy, c, p.D, p.end);
        if constexpr (WHAT != ROWS_PACK) {
            q = *reinterpret_cast<const Raw<VW>*>(p.codes + row * p.ldc + c);
            byte = *act8_scale_at(p.scales, p.lds, row, c);
        }
    };
    if (row < p.M) load(row, piece * VW);
    while (row < p.M) {
        const int64_t r = row;
        const int c = piece * VW;
        const Raw<16> xr = x;
        const Raw<VW> qr = q;
        const float scale = act8_scale(byte);
        row += p.step_rows;
        piece += p.step;
        if (piece >= p.pieces) {
            piece -= p.pieces;
            ++row;
        }
        if (row < p.M) load(row, piece * VW);
        float v[VW];
        if constexpr (WHAT == ROWS_PACK) {
            piece_values<T>(xr, static_cast<const T*>(p.x) + r * p.ldx, c, p.D, p.end, true, v);
            act8_store<T>(v, c, p.Dp, p.codes + r * p.ldc, act8_scale_at(p.scales, p.lds, r, c));
        } else {
            act8_values(qr.w[0], scale, v);
            if constexpr (VW == 8) act8_values(qr.w[1], scale, v + 4);
            T* y = static_cast<T*>(p.y) + r * p.ldy;
            if constexpr (WHAT == ROWS_LEAKY) {
                float g[VW];
                piece_values<T>(xr, y, c, p.D, p.end, true, g);
#pragma unroll
                for (int k = 0; k < VW; ++k) v[k] = v[k] > 0.f ? g[k] : kLeakySlope * g[k];
            }
            piece_store<T>(y, c, p.D, p.end, v);
        }
    }
}

constexpr int kRowsGroups = 8192;   // 32 waves per CU of the launch's stride (2048 .. 16384 measured: 54.7, 53.4, 51.7, 51.6 us on 8192 x 5397)

template <int WHAT>
int launch_rows(const char* what, int type, const RowsParams& p0, pcvae_stream_t stream) {
    RowsParams p = p0;
    if (p.M == 0) return PCVAE_OK;
    p.Dp = (int)cdiv(p.D, kAct8Block) * kAct8Block;
    const int vw = type == PCVAE_ROW_F32 ? 4 : 8;
    p.pieces = p.Dp / vw;
    p.end = row_end(p.D, vw, p.Dp);
    const int64_t groups = cdiv(p.M * p.pieces, 256);
    const dim3 grid((unsigned)(groups < kRowsGroups ? groups : kRowsGroups));
    p.step_rows = (int64_t)grid.x * 256 / p.pieces;
    p.step = (int)((int64_t)grid.x * 256 % p.pieces);
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
// fp16 g is exact in two components, bf16 g in one; behind a norm the factor g r_m is an fp32 number again (three).  Exact means |g| (behind
// a norm |g r_m|) from 2^-110, below which components are too small for a bf16 and vanish one after the other, to 3.39e38, above which the
// first rounds to an infinity; an infinite g makes its row of dW NaN (its db keeps the infinity).
//
// One workgroup: 128 (n) x 64 KT (k) of dW over a range of rows m, four waves of 64 x 32 KT.  Both operands run ALONG the contraction in
// memory's slow direction, so a chunk of 32 rows is turned on its way to LDS: a wave takes 8 consecutive rows, a lane holds 2 (KT)
// neighbouring columns of all 8, and a column's 8 values are the 16-byte operand piece of an MFMA.  LDS image of an operand:
// [4 pieces of 8 rows][i][64 lanes][16 bytes], column = 2 lane + i (KT lane + i): consecutive lanes, consecutive 16 bytes on both sides (no
// conflicts), and a wave whose MFMA tiles are the i of 32 lanes ends with KT neighbouring columns of dW per lane: wide stores.
// Two stages, one barrier per chunk, the loads of two chunks in flight over the products.  Nothing in the loop is a scalar load: its
// wait would be a wait for every LDS read too.
constexpr int TN = 128, TM = 32;
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));

struct DwParams {
    const void* g; int64_t ldg;
    const uint8_t* codes; int64_t ldc; const uint8_t* scales; int64_t lds;
    const float* mean; const float* rstd; const float* w; const float* b;   // the norm's, or null
    int64_t M; int N, K, Kp;
    int nn, nk, nz;            // tiles along n and k, ranges of m
    int64_t m_per;             // rows of a range, a multiple of 2 TM
    float* part;               // nz > 1: [nz][nn nk][TN][TK] partial tiles, [nz][nn TN] partial column sums
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

// two neighbouring values of a gradient row
template <typename T> struct Pair;
template <> struct Pair<float> {
    typedef Raw<8> raw;
    static __device__ __forceinline__ float get(const raw& r, int i) { return __uint_as_float(r.w[i]); }
    static __device__ __forceinline__ raw one(const float* p) { return raw{{__float_as_uint(*p), 0}}; }
};
template <> struct Pair<__bf16> {
    typedef Raw<4> raw;
    static __device__ __forceinline__ float get(const raw& r, int i) { return i ? high2(r.w[0]) : low2(r.w[0]); }
    static __device__ __forceinline__ raw one(const __bf16* p) { return raw{{*reinterpret_cast<const uint16_t*>(p)}}; }
};
template <> struct Pair<_Float16> {
    typedef Raw<4> raw;
    static __device__ __forceinline__ float get(const raw& r, int i) { return (float)__builtin_bit_cast(f16x2_t, r.w[0])[i]; }
    static __device__ __forceinline__ raw one(const _Float16* p) { return raw{{*reinterpret_cast<const uint16_t*>(p)}}; }
};

template <typename T, int NC, bool NORM, int KT>
__global__ __launch_bounds__(256, 2) void act8_weight_kernel(DwParams p) {
    constexpr int TK = 64 * KT;
    __shared__ uint4 sA0[NC][4][TN], sA1[NC][4][TN];
    __shared__ uint4 sB0[4][TK], sB1[4][TK];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // logical order: all tiles of a range of rows next to each other (they share g and the codes in one XCD's L2)
    const int id = xcd_remap(blockIdx.x, gridDim.x);
    const int tiles = p.nn * p.nk, z = id / tiles, tile = id % tiles, tn = tile / p.nk, tk = tile % p.nk;
    const int64_t m0 = (int64_t)z * p.m_per, m1 = m0 + p.m_per < p.M ? m0 + p.m_per : p.M;

    // Columns past the end: the last pair of an odd N is loaded one column early (its second value is the real one: value i of a pair at
    // n0 = N - 1 is column n0 + i - 1); whole pairs past N and codes past Kp read the last ones.  None of those reaches dW.
    const int nc = min(tn * TN + 2 * lane, p.N - 2);
    const int kc = min(tk * TK + KT * lane, p.Kp - KT);
    const T* g = static_cast<const T*>(p.g);
    const bool sums = NORM || (tk == 0 && p.db != nullptr);

    struct Chunk {
        typename Pair<T>::raw g[8];
        uint32_t q[8];
        uint2 s;
        float r, mu;
    };
    float sum[2] = {0.f, 0.f}, muc[2] = {0.f, 0.f};
    const uint32_t goff = (uint32_t)(nc < 0 ? 0 : nc) * (uint32_t)sizeof(T), qoff = (uint32_t)kc;

    // this wave's 8 rows from m on, all inside the range
    auto fetch = [&](int64_t m, Chunk& c) {
        const char* gr = reinterpret_cast<const char*>(g + m * p.ldg);
        const uint8_t* qr = p.codes + m * p.ldc;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            c.g[j] = *reinterpret_cast<const typename Pair<T>::raw*>(gr + goff);
            if constexpr (KT == 4) c.q[j] = *reinterpret_cast<const uint32_t*>(qr + qoff);
            else c.q[j] = *reinterpret_cast<const uint16_t*>(qr + qoff);
            gr += p.ldg * (int64_t)sizeof(T);
            qr += p.ldc;
        }
        c.s = *reinterpret_cast<const uint2*>(p.scales + (m >> 3) * p.lds + (kc >> 5) * 8);   // m is a multiple of 8
        if constexpr (NORM) {
            c.r = p.rstd[m + (lane & 7)];
            c.mu = p.mean[m + (lane & 7)];
        }
    };
    // the same at the range's end (rows from m1 on repeat the last one: place() drops them) and for a single column
    auto fetch_end = [&](int64_t m, Chunk& c) {
#pragma unroll 1
        for (int j = 0; j < 8; ++j) {
            const int64_t mm = m + j < m1 ? m + j : m1 - 1;
            const char* gr = reinterpret_cast<const char*>(g + mm * p.ldg);
            const uint8_t* qr = p.codes + mm * p.ldc;
            typename Pair<T>::raw gv;
            if (p.N > 1) gv = *reinterpret_cast<const typename Pair<T>::raw*>(gr + goff);
            else gv = Pair<T>::one(reinterpret_cast<const T*>(gr));
            uint32_t qv;
            if constexpr (KT == 4) qv = *reinterpret_cast<const uint32_t*>(qr + qoff);
            else qv = *reinterpret_cast<const uint16_t*>(qr + qoff);
#pragma unroll
            for (int i = 0; i < 8; ++i) {   // (no register is indexed by a variable)
                if (i == j) c.g[i] = gv, c.q[i] = qv;
            }
        }
        c.s = *reinterpret_cast<const uint2*>(p.scales + ((m < m1 ? m : m1 - 1) >> 3) * p.lds + (kc >> 5) * 8);
        if constexpr (NORM) {
            const int64_t mm = m + (lane & 7) < m1 ? m + (lane & 7) : m1 - 1;
            c.r = p.rstd[mm];
            c.mu = p.mean[mm];
        }
    };
    // a chunk's 8 rows as operand pieces; rows >= `rows` count nothing (their scale bytes need not be written)
    auto place = [&](const Chunk& c, uint4 (&A)[NC][4][TN], uint4 (&B)[4][TK], auto with_sums, auto at_end, int rows) {
        constexpr bool SUMS = decltype(with_sums)::value, ENDING = decltype(at_end)::value;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            uint4 w[NC];
            if constexpr (std::is_same<T, __bf16>::value && !NORM && !SUMS && !ENDING) {   // the values are their own only component
                const uint32_t sel = i ? 0x07060302u : 0x05040100u;
                w[0] = make_uint4(__builtin_amdgcn_perm(c.g[1].w[0], c.g[0].w[0], sel), __builtin_amdgcn_perm(c.g[3].w[0], c.g[2].w[0], sel),
                                  __builtin_amdgcn_perm(c.g[5].w[0], c.g[4].w[0], sel), __builtin_amdgcn_perm(c.g[7].w[0], c.g[6].w[0], sel));
            } else {
                float v[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    v[j] = Pair<T>::get(c.g[j], i);
                    if constexpr (ENDING) v[j] = j < rows ? v[j] : 0.f;
                }
                if constexpr (SUMS) sum[i] += ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
                if constexpr (NORM) {
                    float t = 0.f;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float r = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(c.r), j));
                        const float mu = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(c.mu), j));
                        v[j] *= r;
                        t = fmaf(v[j], mu, t);
                    }
                    muc[i] += t;
                }
                split8<NC>(v, w);
            }
#pragma unroll
            for (int k = 0; k < NC; ++k) A[k][wave][64 * i + lane] = w[k];
        }
        uint32_t e[8][KT / 2];   // bf16 pairs (columns 2 h, 2 h + 1) of a row
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float s = act8_scale(((j < 4 ? c.s.x : c.s.y) >> (8 * (j & 3))) & 0xffu);
            e[j][0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c.q[j], s, false));
            if constexpr (KT == 4) e[j][1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c.q[j], s, true));
            if constexpr (ENDING) {
#pragma unroll
                for (int h = 0; h < KT / 2; ++h) e[j][h] = j < rows ? e[j][h] : 0u;
            }
        }
#pragma unroll
        for (int h = 0; h < KT / 2; ++h) {
            B[wave][64 * (2 * h) + lane] =
                make_uint4(__builtin_amdgcn_perm(e[1][h], e[0][h], 0x05040100u), __builtin_amdgcn_perm(e[3][h], e[2][h], 0x05040100u),
                           __builtin_amdgcn_perm(e[5][h], e[4][h], 0x05040100u), __builtin_amdgcn_perm(e[7][h], e[6][h], 0x05040100u));
            B[wave][64 * (2 * h + 1) + lane] =
                make_uint4(__builtin_amdgcn_perm(e[1][h], e[0][h], 0x07060302u), __builtin_amdgcn_perm(e[3][h], e[2][h], 0x07060302u),
                           __builtin_amdgcn_perm(e[5][h], e[4][h], 0x07060302u), __builtin_amdgcn_perm(e[7][h], e[6][h], 0x07060302u));
        }
    };

    const int hn = 32 * (wave >> 1), hk = 32 * (wave & 1), l = lane & 31;
    f32x16_t acc[2][KT];
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int b = 0; b < KT; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[a][b][i] = 0.f;
    auto multiply = [&](uint4 (&A)[NC][4][TN], uint4 (&B)[4][TK]) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int piece = 2 * s + (lane >> 5);
            bf16x8_t b[KT];
#pragma unroll
            for (int t = 0; t < KT; ++t) b[t] = __builtin_bit_cast(bf16x8_t, B[piece][64 * t + hk + l]);
#pragma unroll
            for (int k = NC - 1; k >= 0; --k)   // the smallest components first
#pragma unroll
                for (int a = 0; a < 2; ++a) {
                    const bf16x8_t av = __builtin_bit_cast(bf16x8_t, A[k][piece][64 * a + hn + l]);
#pragma unroll
                    for (int t = 0; t < KT; ++t) acc[a][t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(av, b[t], acc[a][t], 0, 0, 0);
                }
        }
    };

    // The order of a half of the loop, for three components: one product, five vector operations of the next chunk's conversion (what a
    // product hides: four or five, measured on two waves per SIMD), the operand reads ahead and the stores behind.  Kernel and
    // join, both sides in turn: 4864 x 1024 over 32768 rows 866 -> 847 us, 1024 x 2048 over 16384 rows 191 -> 188 us, behind a norm 213 -> 205
    // us; with one or two components the compiler's own order is as good.
    auto weave = [&]() {
        if constexpr (NC == 3 && KT == 4) {
            constexpr int PRODUCTS = 4 * NC * KT, READS = KT + 4 * NC - 2, STORES = 2 * NC + KT;
            __builtin_amdgcn_sched_group_barrier(0x100, KT + 2, 0);
#pragma unroll
            for (int i = 0; i < PRODUCTS; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x002, 5, 0);
                if (i < READS) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                if (i >= PRODUCTS - STORES) __builtin_amdgcn_sched_group_barrier(0x200, 1, 0);
            }
        }
    };
    // whole pairs of chunks: no branch between the two barriers, so products and the next chunk's conversion interleave
    const std::integral_constant<bool, true> yes{};
    const std::integral_constant<bool, false> no{};
    const int pairs = p.N > 1 ? (int)((m1 - m0) / (2 * TM)) : 0;
    const int64_t mw = m0 + 8 * wave;
    auto run = [&](auto with_sums) {
        constexpr int AHEAD = KT == 2 ? 2 : 1;   // chunks in flight: the wide tile's accumulators leave registers for one
        Chunk R0, R1v;
        Chunk& R1 = AHEAD == 2 ? R1v : R0;
        const int last = 2 * pairs - 1;
        auto at = [&](int chunk) { return mw + (int64_t)(chunk < last ? chunk : last) * TM; };
        fetch(at(0), R0);
        if (AHEAD == 2) fetch(at(1), R1);
        place(R0, sA0, sB0, with_sums, no, 8);
        fetch(at(AHEAD), R0);
        __syncthreads();
        for (int c = 0; c + 2 < 2 * pairs; c += 2) {
            place(R1, sA1, sB1, with_sums, no, 8);
            fetch(at(c + 1 + AHEAD), R1);
            multiply(sA0, sB0);
            weave();
            __syncthreads();
            place(R0, sA0, sB0, with_sums, no, 8);
            fetch(at(c + 2 + AHEAD), R0);
            multiply(sA1, sB1);
            weave();
            __syncthreads();
        }
        place(R1, sA1, sB1, with_sums, no, 8);
        multiply(sA0, sB0);
        __syncthreads();
        multiply(sA1, sB1);
    };
    if (pairs > 0) {
        if (sums) run(yes);
        else run(no);
    }
    for (int64_t m = m0 + (int64_t)pairs * 2 * TM; m < m1; m += TM) {   // what is left of the range
        Chunk R;
        fetch_end(m + 8 * wave, R);
        __syncthreads();
        const int64_t left = m1 - m - 8 * wave;
        place(R, sA0, sB0, yes, yes, left < 8 ? (int)left : 8);
        __syncthreads();
        multiply(sA0, sB0);
    }
    __syncthreads();

    float (*sSum)[4][TN] = reinterpret_cast<float (*)[4][TN]>(&sA0[0][0][0]);   // column sums, behind the last product
    if (sums) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            sSum[0][wave][64 * i + lane] = sum[i];
            if constexpr (NORM) sSum[1][wave][64 * i + lane] = muc[i];
        }
        __syncthreads();
    }
    auto total = [&](int which, int at) { return (sSum[which][0][at] + sSum[which][1][at]) + (sSum[which][2][at] + sSum[which][3][at]); };
    if (tk == 0 && p.db != nullptr && threadIdx.x < TN) {
        const int i = threadIdx.x >> 6, n0 = tn * TN + 2 * lane, n = n0 + i - (n0 == p.N - 1 && p.N > 1);
        if (n >= n0 && n < p.N) {
            const float t = total(0, threadIdx.x);
            if (p.nz > 1) p.part_db[(int64_t)z * p.nn * TN + n] = t;
            else p.db[n] = p.accumulate ? p.db[n] + t : t;
        }
    }
    const int kk = KT * (hk + l), k = tk * TK + kk;   // KT neighbouring columns
    float wv[KT], bv[KT];
    if constexpr (NORM) {
#pragma unroll
        for (int t = 0; t < KT; ++t) {
            wv[t] = p.w && k + t < p.K ? p.w[k + t] : 1.f;
            bv[t] = p.b && k + t < p.K ? p.b[k + t] : 0.f;
        }
    }
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int pair = hn + (i & 3) + 8 * (i >> 2) + 4 * (lane >> 5), n0 = tn * TN + 2 * pair;
            const int n = n0 + a - (n0 == p.N - 1 && p.N > 1);
            float v[KT];
#pragma unroll
            for (int t = 0; t < KT; ++t) v[t] = acc[a][t][i];
            if constexpr (NORM) {
                const float c0 = total(0, 64 * a + pair), c1 = total(1, 64 * a + pair);
#pragma unroll
                for (int t = 0; t < KT; ++t) v[t] = fmaf(wv[t], v[t] - c1, bv[t] * c0);
            }
            if (n < n0 || n >= p.N) continue;
            float* out = p.nz > 1 ? p.part + (((int64_t)z * tiles + tile) * TN + (n - tn * TN)) * TK + kk : p.dW + (int64_t)n * p.lddw + k;
            const bool add = p.nz == 1 && p.accumulate;
            if (p.nz > 1 || k + KT <= p.K) {
                Raw<4 * KT> r;
                if (add) r = *reinterpret_cast<const Raw<4 * KT>*>(out);
#pragma unroll
                for (int t = 0; t < KT; ++t) r.w[t] = __float_as_uint(add ? __uint_as_float(r.w[t]) + v[t] : v[t]);
                *reinterpret_cast<Raw<4 * KT>*>(out) = r;
            } else {
#pragma unroll
                for (int t = 0; t < KT; ++t)
                    if (k + t < p.K) out[t] = add ? out[t] + v[t] : v[t];
            }
        }
}

// The ranges of rows joined: SL neighbouring runs of ranges per value, added in order (the same bits every run).  64 float4 of a tile per
// SL threads; four ranges in flight per thread.
template <int SL>
__global__ __launch_bounds__(256) void act8_weight_join_kernel(DwParams p, int TK) {
    __shared__ f32x4_t sh[256];
    const int sum_groups = p.db ? (p.N + 31) / 32 : 0;
    if ((int)blockIdx.x < sum_groups) {   // 32 column sums, 8 runs of ranges each
        float* part = reinterpret_cast<float*>(sh);
        const int n = blockIdx.x * 32 + (threadIdx.x & 31), run = threadIdx.x >> 5, per = (p.nz + 7) / 8;
        const int z0 = run * per, z1 = z0 + per < p.nz ? z0 + per : p.nz;
        float s = 0.f;
        if (n < p.N) {
            for (int z = z0; z < z1; z += 8) {
                float v[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = z + j < z1 ? p.part_db[(int64_t)(z + j) * p.nn * TN + n] : 0.f;
#pragma unroll
                for (int j = 0; j < 8; ++j) s += v[j];
            }
        }
        part[threadIdx.x] = s;
        __syncthreads();
        if (run == 0 && n < p.N) {
#pragma unroll
            for (int r = 1; r < 8; ++r) s += part[r * 32 + threadIdx.x];
            p.db[n] = p.accumulate ? p.db[n] + s : s;
        }
        return;
    }
    const int block = blockIdx.x - sum_groups, blocks = gridDim.x - sum_groups;
    const int tiles = p.nn * p.nk, per_tile = TN * TK / 4, cols = 256 / SL;
    const int64_t total = (int64_t)tiles * per_tile;
    const int slice = threadIdx.x / cols, at = threadIdx.x % cols;
    const int per = (p.nz + SL - 1) / SL, z0 = slice * per, z1 = z0 + per < p.nz ? z0 + per : p.nz;
    for (int64_t i0 = (int64_t)block * cols; i0 < total; i0 += (int64_t)blocks * cols) {   // total is a multiple of cols
        const int64_t i = i0 + at;
        const int tile = (int)(i / per_tile), e = (int)(i % per_tile) * 4;
        const int n = tile / p.nk * TN + e / TK, k = tile % p.nk * TK + e % TK;
        const bool inside = n < p.N && k < p.K;
        f32x4_t s = {0.f, 0.f, 0.f, 0.f};
        if (inside) {
            const float* q = p.part + (int64_t)tile * TN * TK + e;
            const int64_t hop = (int64_t)tiles * TN * TK;
            for (int z = z0; z < z1; z += 4) {
                f32x4_t v[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    v[j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
                    if (z + j < z1) v[j] = *reinterpret_cast<const f32x4_t*>(q + (z + j) * hop);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) s += v[j];
            }
        }
        if constexpr (SL > 1) {
            __syncthreads();
            sh[threadIdx.x] = s;
            __syncthreads();
#pragma unroll
            for (int j = 1; j < SL; ++j) s += sh[j * cols + at];   // (slice 0 keeps the sum of all)
        }
        if (slice == 0 && inside) {
            float* out = p.dW + (int64_t)n * p.lddw + k;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (k + j < p.K) out[j] = p.accumulate ? out[j] + s[j] : s[j];
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

// Tile width and ranges of rows.  The wide tile (128 x 256) converts less per product, the narrow one (128 x 128) has two chunks in flight
// and half the partial tile per range: measured on 8192 rows, us of 128 / 256 columns: 256 x 256 24 / 27, 256 x 1419 43 / 42, 1152 x 256
// 38 / 37; on 16384 rows 1024 x 2048 245 / 212; 32768 rows 4864 x 1024 1120 / 905.  It is taken from 2048 chunks of 32 rows on, over all tiles -
// all of these at widths that both tiles pad alike; the rule does not look at padding (K in 257 .. 384 computes 512 columns where the narrow
// tile would compute 384: 1024 x 300 over 16384 rows 67 us).
// Ranges: the fewest rounds of 512 resident workgroups, a chunk's time against the partial tiles' traffic (flat: within 5 % over a factor
// of two in the number of ranges), 64 at most: one or two tiles over a long batch do not fill the chip (65536 rows: 128 x 257 61 us, 16 x
// 256 57 us).  A single column (N = 1) takes every chunk the way a range's last one goes: 65536 rows, K = 200 111 us.
struct DwPlan { int kt, nn, nk, nz; int64_t m_per; };
DwPlan dw_plan(int64_t M, int64_t N, int64_t K) {
    DwPlan d;
    const int64_t chunks = cdiv(M, TM);
    d.kt = K > 128 && cdiv(N, TN) * cdiv(K, 256) * chunks >= 2048 ? 4 : 2;
    d.nn = (int)cdiv(N, TN);
    d.nk = (int)cdiv(K, 64 * d.kt);
    const int64_t tiles = (int64_t)d.nn * d.nk;
    double best = 0.;
    int64_t pick = 1;
    for (int64_t nz = 1; nz <= 64 && nz * 2 <= chunks + 1; ++nz) {
        const double rounds = (double)cdiv(tiles * nz, 512);
        const double cost = rounds * ((double)cdiv(chunks, nz) + 4.) + (nz > 1 ? 6. + (double)tiles * nz * 64 * d.kt / (1 << 13) : 0.);
        if (nz == 1 || cost < best) best = cost, pick = nz;
    }
    d.m_per = cdiv(cdiv(M, pick), 2 * TM) * 2 * TM;
    d.nz = (int)cdiv(M, d.m_per);
    return d;
}
size_t dw_ws(const DwPlan& d) {
    return d.nz > 1 ? ((size_t)d.nz * d.nn * d.nk * TN * 64 * d.kt + (size_t)d.nz * d.nn * TN) * sizeof(float) : 0;
}

template <typename T, int NC, int KT>
void launch_dw_tile(const DwParams& p, pcvae_stream_t stream) {
    const dim3 grid((unsigned)(p.nn * p.nk * p.nz));
    if (p.mean)
        hipLaunchKernelGGL((act8_weight_kernel<T, 3, true, KT>), grid, dim3(256), 0, as_stream(stream), p);
    else
        hipLaunchKernelGGL((act8_weight_kernel<T, NC, false, KT>), grid, dim3(256), 0, as_stream(stream), p);
}
template <typename T, int NC>
int launch_dw(const DwParams& p, int kt, pcvae_stream_t stream) {
    if (kt == 4) launch_dw_tile<T, NC, 4>(p, stream);
    else launch_dw_tile<T, NC, 2>(p, stream);
    if (int rc = check_launch("act8_bwd_weight")) return rc;
    if (p.nz == 1) return PCVAE_OK;
    const int64_t vecs = (int64_t)p.nn * p.nk * TN * 64 * kt / 4;
    const int64_t sums = p.db ? cdiv(p.N, 32) : 0;
    auto grid_of = [&](int cols) { return dim3((unsigned)(sums + (cdiv(vecs, cols) < 4096 ? cdiv(vecs, cols) : 4096))); };
    if (p.nz >= 8)
        hipLaunchKernelGGL(act8_weight_join_kernel<8>, grid_of(32), dim3(256), 0, as_stream(stream), p, 64 * kt);
    else
        hipLaunchKernelGGL(act8_weight_join_kernel<1>, grid_of(256), dim3(256), 0, as_stream(stream), p, 64 * kt);
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
    p.part_db = need ? p.part + (size_t)d.nz * d.nn * d.nk * TN * 64 * d.kt : nullptr;
    if (type == PCVAE_ROW_F32) return launch_dw<float, 3>(p, d.kt, stream);
    if (type == PCVAE_ROW_BF16) return launch_dw<__bf16, 1>(p, d.kt, stream);
    return launch_dw<_Float16, 2>(p, d.kt, stream);
}
