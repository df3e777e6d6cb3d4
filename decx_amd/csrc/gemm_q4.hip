// Products with weights held in 4 bits:
//
//   Y (M x N) = X (M x K) . W^T,   W(n, k) = (code(n, k) - zero(n, g)) * scale(n, g),   g = k / group
//
// X in fp16, or in int8 with a factor per row.  A code less its zero point is a whole number of -15..15: exact in fp16 and
// in int8.  The matrix instruction therefore multiplies X by whole numbers, group by group, and only the sum of a group is
// multiplied by its scale, in fp32: no product of code and scale is ever rounded to 16 bits.
#include "gemm_q4.hpp"
#include "split_k_exchange.hpp"

namespace decx_hip {

namespace {

typedef _Float16 halfx2 __attribute__((ext_vector_type(2)));
typedef int intx4 __attribute__((ext_vector_type(4)));
typedef halfx8 halfx8_u __attribute__((aligned(2)));      // 16 bytes of X at any element: the hardware takes them unaligned
typedef uintx2 uintx2_u __attribute__((aligned(1)));

__device__ __forceinline__ halfx2 as_half2(uint32_t w) { return __builtin_bit_cast(halfx2, w); }

// Eight codes of a word less the zero point, as fp16.  A code in the low bits of 0x6400 reads 1024 + code, in bits 4..7
// 1024 + 16 code; both steps back are exact in fp16.
struct ZeroF16 { halfx2 low, high; };                     // -(1024 + zero), -(64 + zero), twice each
__device__ __forceinline__ ZeroF16 zero_f16(uint32_t z)
{
    const _Float16 low = (_Float16)(float)-(int)(1024 + z), high = (_Float16)(float)-(int)(64 + z);
    return {halfx2{low, low}, halfx2{high, high}};
}
__device__ __forceinline__ halfx8 widen_f16(uint32_t w, const ZeroF16& z)
{
    const halfx2 sixteenth = {(_Float16)0.0625f, (_Float16)0.0625f};
    const uint32_t v = w >> 8;
    const halfx2 a = as_half2((w & 0x000f000fu) | 0x64006400u) + z.low;
    const halfx2 b = __builtin_elementwise_fma(as_half2((w & 0x00f000f0u) | 0x64006400u), sixteenth, z.high);
    const halfx2 c = as_half2((v & 0x000f000fu) | 0x64006400u) + z.low;
    const halfx2 d = __builtin_elementwise_fma(as_half2((v & 0x00f000f0u) | 0x64006400u), sixteenth, z.high);
    return halfx8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
// The same as int8, columns in the order 0, 4, 1, 5 | 2, 6, 3, 7.  zero: the zero point in every byte.
__device__ __forceinline__ uintx2 widen_i8(uint32_t w, uint32_t zero)
{
    const uint32_t low = ((w & 0x0f0f0f0fu) | 0x80808080u) - zero, high = (((w >> 4) & 0x0f0f0f0fu) | 0x80808080u) - zero;
    return uintx2{low ^ 0x80808080u, high ^ 0x80808080u};
}
// Eight int8 of X in that order.
__device__ __forceinline__ uintx2 order_i8(uintx2 x)
{
    return uintx2{__builtin_amdgcn_perm(x[1], x[0], 0x05010400u), __builtin_amdgcn_perm(x[1], x[0], 0x07030602u)};
}

// Columns k..k+7 of a row of X, zero from K on.
__device__ __forceinline__ halfx8 load_x8(const _Float16* row, uint32_t k, uint32_t K)
{
    if (k + 8 <= K) return *(const halfx8_u*)(row + k);
    halfx8 v = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < 8; ++e) if (k + e < K) v[e] = row[k + e];
    return v;
}
__device__ __forceinline__ uintx2 load_x8(const signed char* row, uint32_t k, uint32_t K)
{
    if (k + 8 <= K) return *(const uintx2_u*)(row + k);
    uintx2 v = {0, 0};
#pragma unroll
    for (int e = 0; e < 8; ++e) if (k + e < K) v[e / 4] |= (uint32_t)(unsigned char)row[k + e] << (8 * (e % 4));
    return v;
}

template <int GPB> struct Scales { typedef _Float16 type __attribute__((ext_vector_type(GPB))); };
template <> struct Scales<1> { typedef _Float16 type; };
template <int GPB> struct Zeros { typedef uint32_t type; };
template <> struct Zeros<1> { typedef uint8_t type; };
template <> struct Zeros<2> { typedef uint16_t type; };

__device__ __forceinline__ void store_y(const GemmQ4Args& g, uint32_t m, uint32_t n, float v)
{
    if (g.x_scales) v *= g.x_scales[m];
    if (g.C) {
        const size_t at = (size_t)m * g.ldc + n;
        const float c = g.y_f32 ? ((const float*)g.C)[at] : (float)((const _Float16*)g.C)[at];
        v = __builtin_fmaf(c, g.beta, g.alpha * v);
    }
    const size_t at = (size_t)m * g.ldy + n;
    if (g.y_f32) ((float*)g.Y)[at] = v;
    else ((_Float16*)g.Y)[at] = (_Float16)v;
}

}  // namespace

// A workgroup owns T row tiles of W (16 T columns of Y) and 16 TM rows of X; its wavefronts deal the column tiles of W among
// themselves and their sums meet in LDS, in wavefront order.  GPB: groups per column tile (128 / group).
template <bool I8, int GPB, int TM, int T, int WAVES>
__global__ void __launch_bounds__(WAVES * 64)
gemm_q4_rows_kernel(const GemmQ4Args g)
{
    typedef typename std::conditional<I8, signed char, _Float16>::type X_t;
    __shared__ float red[WAVES][T * TM][4][64];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, l16 = lane & 15, kg = lane >> 4;
    const uint32_t tile0 = blockIdx.x * T, m0 = blockIdx.y * (16 * TM);

    const X_t* row[TM];
    bool has[TM];
#pragma unroll
    for (int i = 0; i < TM; ++i) {
        const uint32_t m = m0 + 16 * i + l16;
        has[i] = m < g.M;
        row[i] = (const X_t*)g.X + (size_t)(has[i] ? m : 0) * g.ldx;
    }
    floatx4 acc[T][TM];
#pragma unroll
    for (int c = 0; c < T; ++c)
#pragma unroll
        for (int i = 0; i < TM; ++i) acc[c][i] = floatx4{0, 0, 0, 0};

    for (uint32_t kt = wave; kt < g.k_tiles; kt += WAVES) {
        const uint32_t k0 = kt * kQ4TileCols + 8 * kg;
        halfx8 xf[TM][4];
        uintx2 xi[TM][4];
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (I8) {
                    xi[i][j] = uintx2{0, 0};
                    if (has[i]) xi[i][j] = order_i8(load_x8(row[i], k0 + 32 * j, g.K));
                } else {
                    xf[i][j] = halfx8{0, 0, 0, 0, 0, 0, 0, 0};
                    if (has[i]) xf[i][j] = load_x8(row[i], k0 + 32 * j, g.K);
                }
            }
#pragma unroll
        for (int c = 0; c < T; ++c) {
            const uint32_t nt = tile0 + c < g.n_tiles ? tile0 + c : g.n_tiles - 1;
            const size_t tile = (size_t)nt * g.k_tiles + kt;
            const uintx4 w = *(const uintx4*)(g.codes + tile * kQ4TileBytes + lane * 16);
            const size_t at = (tile * 16 + l16) * GPB;
            const typename Scales<GPB>::type sv = *(const typename Scales<GPB>::type*)(g.scales + at);
            uint32_t zv = 0x08080808u;
            if (g.zeros) zv = *(const typename Zeros<GPB>::type*)(g.zeros + at);
#pragma unroll
            for (int q = 0; q < GPB; ++q) {
                constexpr int STEPS = 4 / GPB;             // words of a group
                float s;
                if constexpr (GPB == 1) s = (float)sv; else s = (float)sv[q];
                if (kt * kQ4TileCols + q * (kQ4TileCols / GPB) >= g.K) s = 0.f;       // a group beyond the last column
                const uint32_t z = (zv >> (8 * q)) & 0xffu;
                if constexpr (I8) {
                    const uint32_t zz = z * 0x01010101u;
#pragma unroll
                    for (int i = 0; i < TM; ++i) {
                        intx4 part = {0, 0, 0, 0};
                        if constexpr (STEPS == 1) {
                            part = __builtin_amdgcn_mfma_i32_16x16x32_i8(__builtin_bit_cast(long, xi[i][q]), __builtin_bit_cast(long, widen_i8(w[q], zz)), part, 0, 0, 0);
                        } else {
#pragma unroll
                            for (int j = q * STEPS; j < (q + 1) * STEPS; j += 2) {
                                const uintx2 w0 = widen_i8(w[j], zz), w1 = widen_i8(w[j + 1], zz);
                                const intx4 a = {(int)xi[i][j][0], (int)xi[i][j][1], (int)xi[i][j + 1][0], (int)xi[i][j + 1][1]};
                                const intx4 b = {(int)w0[0], (int)w0[1], (int)w1[0], (int)w1[1]};
                                part = __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, part, 0, 0, 0);
                            }
                        }
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[c][i][e] = __builtin_fmaf((float)part[e], s, acc[c][i][e]);
                    }
                } else {
                    const ZeroF16 zz = zero_f16(z);
#pragma unroll
                    for (int i = 0; i < TM; ++i) {
                        floatx4 part = {0, 0, 0, 0};
#pragma unroll
                        for (int j = q * STEPS; j < (q + 1) * STEPS; ++j)
                            part = __builtin_amdgcn_mfma_f32_16x16x32_f16(xf[i][j], widen_f16(w[j], zz), part, 0, 0, 0);
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[c][i][e] = __builtin_fmaf(part[e], s, acc[c][i][e]);
                    }
                }
            }
        }
    }
    // lane (kg, l16) holds rows 4 kg .. 4 kg + 3 of X and row l16 of W of every 16 x 16 piece
#pragma unroll
    for (int c = 0; c < T; ++c)
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) red[wave][c * TM + i][e][lane] = acc[c][i][e];
    __syncthreads();
    for (int o = t; o < T * TM * 256; o += WAVES * 64) {
        const int piece = o / 256, m_in = (o / 16) % 16, n_in = o % 16;
        const uint32_t m = m0 + 16 * (piece % TM) + m_in, n = (tile0 + piece / TM) * 16 + n_in;
        if (m >= g.M || n >= g.N) continue;
        float v = 0;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) v += red[w][piece][m_in % 4][(m_in / 4) * 16 + n_in];
        store_y(g, m, n, v);
    }
}

namespace {

template <bool I8, int GPB> int launch_as(const GemmQ4Args& g, hipStream_t stream)
{
    constexpr int TM = 1, T = 1, WAVES = 8;
    // (the grid's second dimension holds 65 535 workgroups: longer ones go in several launches)
    constexpr uint32_t ROWS = 16 * TM, MOST = 65535;
    for (uint32_t m0 = 0; m0 < g.M; m0 += MOST * ROWS) {
        GemmQ4Args a = g;
        a.X = (const char*)g.X + (size_t)m0 * g.ldx * (I8 ? 1 : 2);
        if (g.x_scales) a.x_scales = g.x_scales + m0;
        if (g.C) a.C = (const char*)g.C + (size_t)m0 * g.ldc * (g.y_f32 ? 4 : 2);
        a.Y = (char*)g.Y + (size_t)m0 * g.ldy * (g.y_f32 ? 4 : 2);
        a.M = g.M - m0 < MOST * ROWS ? g.M - m0 : MOST * ROWS;
        hipLaunchKernelGGL((gemm_q4_rows_kernel<I8, GPB, TM, T, WAVES>), dim3((g.n_tiles + T - 1) / T, (a.M + ROWS - 1) / ROWS), dim3(WAVES * 64), 0, stream, a);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return (int)e;
        if (g.M - m0 <= MOST * ROWS) break;
    }
    return 0;
}

}  // namespace

int launch_gemm_q4(bool i8, uint32_t group, const GemmQ4Args& g, hipStream_t stream)
{
    switch (group) {
    case 128: return i8 ? launch_as<true, 1>(g, stream) : launch_as<false, 1>(g, stream);
    case 64:  return i8 ? launch_as<true, 2>(g, stream) : launch_as<false, 2>(g, stream);
    default:  return i8 ? launch_as<true, 4>(g, stream) : launch_as<false, 4>(g, stream);
    }
}

}  // namespace decx_hip
