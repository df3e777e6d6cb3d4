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
// 1024 + 16 code; the steps back are exact in fp16, and so are their constants: -(1024 + zero) is 0xe400 + zero,
// -(64 + zero) 0xd400 + 16 zero.  (The masks are kept in registers: from there mask and exponent are one instruction.)
struct WidenF16 {
    uint32_t first, second, exponent;
    __device__ __forceinline__ WidenF16() : first(0x000f000fu), second(0x00f000f0u), exponent(0x64006400u)
    {
        asm("" : "+s"(first), "+s"(second), "+v"(exponent));
    }
    struct Zero { halfx2 low, high; };
    static __device__ __forceinline__ Zero zero(uint32_t z) { return {as_half2(z * 0x00010001u + 0xe400e400u), as_half2(z * 0x00100010u + 0xd400d400u)}; }
    __device__ __forceinline__ halfx8 operator()(uint32_t w, const Zero& z) const
    {
        const halfx2 sixteenth = {(_Float16)0.0625f, (_Float16)0.0625f};
        const uint32_t v = w >> 8;
        const halfx2 a = as_half2((w & first) | exponent) + z.low;
        const halfx2 b = __builtin_elementwise_fma(as_half2((w & second) | exponent), sixteenth, z.high);
        const halfx2 c = as_half2((v & first) | exponent) + z.low;
        const halfx2 d = __builtin_elementwise_fma(as_half2((v & second) | exponent), sixteenth, z.high);
        return halfx8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
    }
};
// The same as int8, columns in the order 0, 4, 1, 5 | 2, 6, 3, 7.  With zero points (in every byte of `zero`): code - zero.
// Without: 16 (code - 8), the code in the upper half of its byte (FACTOR, taken back with the scale).
template <bool ZEROS> struct WidenI8 {
    uint32_t mask, sign;
    __device__ __forceinline__ WidenI8() : mask(ZEROS ? 0x0f0f0f0fu : 0xf0f0f0f0u), sign(ZEROS ? 0x80808080u : 0x88888888u)
    {
        asm("" : "+s"(mask), "+v"(sign));
    }
    __device__ __forceinline__ uintx2 operator()(uint32_t w, uint32_t zero) const
    {
        if constexpr (ZEROS) {
            const uint32_t low = ((w & mask) | sign) - zero, high = (((w >> 4) & mask) | sign) - zero;
            return uintx2{low ^ sign, high ^ sign};
        } else {
            const uint32_t v = w ^ sign;
            return uintx2{(v << 4) & mask, v & mask};
        }
    }
};
template <bool I8, bool ZEROS> struct Factor { static constexpr float value = I8 && !ZEROS ? 0.0625f : 1.f; };
// Eight int8 of X in that order.
__device__ __forceinline__ uintx2 order_i8(uintx2 x)
{
    return uintx2{__builtin_amdgcn_perm(x[1], x[0], 0x05010400u), __builtin_amdgcn_perm(x[1], x[0], 0x07030602u)};
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

// Four adjacent outputs of a row, the first of them inside.
__device__ __forceinline__ void store_y4(const GemmQ4Args& g, uint32_t m, uint32_t n, floatx4 v)
{
    if (n + 4 > g.N || !g.quads_ok) {
#pragma unroll
        for (int e = 0; e < 4; ++e) if (n + e < g.N) store_y(g, m, n + e, v[e]);
        return;
    }
    if (g.x_scales) {
        const float s = g.x_scales[m];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] *= s;
    }
    if (g.C) {
        const size_t at = (size_t)m * g.ldc + n;
        floatx4 c;
        if (g.y_f32) {
            c = *(const floatx4*)((const float*)g.C + at);
        } else {
            const halfx4 h = *(const halfx4*)((const _Float16*)g.C + at);
            c = floatx4{(float)h[0], (float)h[1], (float)h[2], (float)h[3]};
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = __builtin_fmaf(c[e], g.beta, g.alpha * v[e]);
    }
    const size_t at = (size_t)m * g.ldy + n;
    if (g.y_f32) *(floatx4*)((float*)g.Y + at) = v;
    else *(halfx4*)((_Float16*)g.Y + at) = halfx4{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
}

}  // namespace

// X in LDS: rows of one column tile of W, 128 columns.  fp16: 256 bytes, 16-byte chunk c (columns 8 c ..) of row r in slot
// c ^ (r % 16).  int8: 128 bytes, chunk 4 s + kg holding the two pieces of 8 columns from 64 s + 8 kg and from 64 s + 32 + 8 kg,
// each in the codes' order, in slot chunk ^ (r / 2 % 8).  So a lane's operand of a matrix instruction is one 16-byte read, and
// the 16 rows that a quarter of a wavefront reads together cover all banks.
template <bool I8> struct XRows {
    static constexpr int BYTES = I8 ? 128 : 256, CHUNKS = BYTES / 16;
    // where the 16 bytes `at` (of CHUNKS, in the order of memory) of a row go
    static __device__ __forceinline__ uint32_t place(int row, int at)
    {
        if constexpr (I8) {
            // their two pieces of 8 columns belong to block j = at / 2 of 32 columns and to kg = at % 2 * 2 + (0, 1); s = j / 2, half j % 2
            const int chunk = at / 4 * 4 + at % 2 * 2;
            return row * BYTES + ((chunk ^ ((row >> 1) & 7)) * 16) + (at / 2 % 2) * 8;
        } else {
            return row * BYTES + ((at ^ (row & 15)) * 16);
        }
    }
    static __device__ __forceinline__ void put(unsigned char* lds, uint32_t place, const uintx4& v)
    {
        if constexpr (I8) {
            // (the second piece's chunk is the next one: the first is even, so its slot differs in the lowest bit)
            *(uintx2*)(lds + place) = order_i8(uintx2{v[0], v[1]});
            *(uintx2*)(lds + (place ^ 16)) = order_i8(uintx2{v[2], v[3]});
        } else {
            *(uintx4*)(lds + place) = v;
        }
    }
    // chunk: 4 j + kg (fp16, step j of 32 columns), 4 s + kg (int8, step s of 64); row16: the row in its tile of 16
    static __device__ __forceinline__ uint32_t slot(int chunk, int row16) { return (chunk ^ (I8 ? (row16 >> 1) & 7 : row16)) * 16; }
};

// ---- few rows --------------------------------------------------------------------------------------------------------
//
// A workgroup owns T row tiles of W (16 T columns of Y) and 16 TM rows of X; its wavefronts deal the column tiles of W among
// themselves and their sums meet in LDS, in wavefront order.  The codes go straight into the registers the matrix instruction
// reads, 1 KB of a tile a load, one step ahead of the products.  X comes out of the L2, where every wavefront reads other
// columns of it.  Read in the instruction's order, 16 rows of 64 bytes a load, it would keep the L1 busy with lines; so a
// wavefront loads whole rows (4 of 256 bytes at a time) and turns them around in LDS of its own, which nobody waits for
// (when it came in: 7 x 5003 x 7001 20.6 -> 8.1 us, 32 x 8192 x 8192 18.5 -> 12.1).  The same of loads under no condition: 1 x 65536
// x 8192 in groups of 32 60 -> 55 us, 1 x 4096 x 16384 8.9 -> 7.5, 60 x 8192 x 4096 int8 10.2 -> 9.2; 17 x 5003 x 7001, where the
// rows are not aligned and half of the loads have none, 13.0 -> 13.6.
// Now (calls; recorded and replayed they take the same, but for the smallest): 1 x 65536 x 8192 in groups of 32 53 us = 5.7 TB/s, the
// codes' way out of HBM; 1 x 8192 x 8192 int8 7.5, 16 x 8192 x 8192 8.7, 7 x 5003 x 7001 7.7, 60 x 8192 x 4096 int8 9.1, 32 x 8192 x 8192
// 11.7, 17 x 5003 x 7001 12.4: the launch (a kernel with nothing to do takes 1.8) and the latency of a wavefront's few column tiles,
// one after the other, loads one step ahead; it waits 35 to 60 % of its time, while neither the vector pipe (24-46 % busy) nor the
// L1 (0.2-0.5 accesses a cycle and CU) nor HBM is full.  1 x 4096 x 4096 takes 4.3 us traced and 3.5 from launch to launch in a
// recorded graph; a call from Python, 5.0, is bound by the host.
template <bool I8, int GPB, bool ZEROS, int TM, int T, int WAVES, int CH>
__global__ void __launch_bounds__(WAVES * 64)
__attribute__((amdgpu_waves_per_eu(TM == 1 ? 4 : 2)))
gemm_q4_rows_kernel(const GemmQ4Args g)
{
    typedef typename std::conditional<I8, signed char, _Float16>::type X_t;
    typedef typename std::conditional<I8, intx4, floatx4>::type P_t;
    typedef typename Scales<GPB>::type S_t;
    typedef XRows<I8> R;
    constexpr int TURN_BYTES = CH * 1024, ROWS_AT_ONCE = 64 / R::CHUNKS, ROWS = CH * ROWS_AT_ONCE;
    constexpr bool AHEAD_ALWAYS = CH <= 8;
    static_assert(ROWS == 16 * TM || (TM == 1 && ROWS < 16 && (ROWS & (ROWS - 1)) == 0), "rows that are held");
    constexpr int RED_BYTES = WAVES * T * TM * 1024;
    __shared__ __attribute__((aligned(1024))) unsigned char lds[WAVES * TURN_BYTES > RED_BYTES ? WAVES * TURN_BYTES : RED_BYTES];
    float (*const red)[T * TM][4][64] = (float (*)[T * TM][4][64])lds;
    const int t = threadIdx.x, lane = t & 63, l16 = lane & 15, kg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const uint32_t tile0 = blockIdx.x * T, m0 = blockIdx.y * (16 * TM);

    unsigned char* const turn = lds + wave * TURN_BYTES;
    // CH loads of ROWS_AT_ONCE rows each.  They and those of the codes are asked for under no condition: behind a branch the
    // compiler cannot tell a load's wait from that for the loads behind it.  Lanes without a row repeat the last one, loads
    // without a row read the first codes, and the last whole column tile is read again where none follows (the columns of a
    // part of a tile are fetched as they are turned).  64 rows of fp16 have no registers for the addresses: there as it was.
    const int turn_row = lane / R::CHUNKS, turn_at = lane % R::CHUNKS;
    const uint32_t here = g.M - m0 < (uint32_t)ROWS ? g.M - m0 : (uint32_t)ROWS, full = here / ROWS_AT_ONCE, rest = here % ROWS_AT_ONCE;
    const uint32_t whole = g.K / kQ4TileCols;
    const auto row_at = [&](uint32_t r) __attribute__((always_inline)) { return (const unsigned char*)g.X + (size_t)(m0 + r) * g.ldx * sizeof(X_t); };
    const unsigned char* const turn_src = AHEAD_ALWAYS && !whole ? g.codes : row_at((uint32_t)turn_row < here ? turn_row : 0);
    const unsigned char* const rest_src = whole && rest ? row_at((uint32_t)turn_row < rest ? turn_row : rest - 1) : turn_src;
    const size_t turn_step = AHEAD_ALWAYS && !whole ? 0 : (size_t)ROWS_AT_ONCE * g.ldx * sizeof(X_t);
    uintx4 turning[CH];
    const auto fetch_rows = [&](uint32_t kt) __attribute__((always_inline)) {
        if constexpr (!AHEAD_ALWAYS) {
            const unsigned char* const src = turn_src + ((size_t)kt * R::BYTES + turn_at * 16);
            if ((kt + 1) * kQ4TileCols <= g.K)
#pragma unroll
                for (int c = 0; c < CH; ++c)
                    if ((uint32_t)(turn_row + c * ROWS_AT_ONCE) < here) __builtin_memcpy(&turning[c], src + c * turn_step, 16);
            return;
        }
        const size_t from = (size_t)(kt < whole ? kt : whole ? whole - 1 : 0) * R::BYTES + turn_at * 16;
#pragma unroll
        for (uint32_t c = 0; c < (uint32_t)CH; ++c) {
            const bool last = c == full && rest;
            const unsigned char* src = g.codes;
            if (c < full) src = turn_src + (from + c * turn_step);
            if (last) src = rest_src + (from + c * turn_step);
            __builtin_memcpy(&turning[c], src, 16);
        }
    };
    const auto turn_rows = [&](uint32_t kt) __attribute__((always_inline)) {
        wavefront_order();
        if ((kt + 1) * kQ4TileCols <= g.K) {
#pragma unroll
            for (int c = 0; c < CH; ++c) R::put(turn, R::place(turn_row + c * ROWS_AT_ONCE, turn_at), turning[c]);
        } else {
#pragma unroll 1
            for (int c = 0; c < CH; ++c)
                if (m0 + turn_row + c * ROWS_AT_ONCE < g.M)
                    R::put(turn, R::place(turn_row + c * ROWS_AT_ONCE, turn_at),
                           load_end((const X_t*)(AHEAD_ALWAYS ? row_at(turn_row + c * ROWS_AT_ONCE) : turn_src + c * turn_step),
                                    kt * kQ4TileCols + turn_at * (16 / sizeof(X_t)), g.K));
        }
        wavefront_order();
    };

    const int held = ROWS < 16 ? l16 & (ROWS - 1) : l16;       // (of fewer rows than 16 the same ones again: they are not stored)
    size_t tile_at[T];
#pragma unroll
    for (int c = 0; c < T; ++c) tile_at[c] = (size_t)(tile0 + c < g.n_tiles ? tile0 + c : g.n_tiles - 1) * g.k_tiles;

    struct Codes { uintx4 w[T]; S_t s[T]; uint32_t z[T]; };
    const auto fetch_codes = [&](Codes& f, uint32_t kt) __attribute__((always_inline)) {
#pragma unroll
        for (int c = 0; c < T; ++c) {
            const size_t tile = tile_at[c] + kt;
            f.w[c] = *(const uintx4*)(g.codes + tile * kQ4TileBytes + lane * 16);
            f.s[c] = *(const S_t*)(g.scales + (tile * 16 + l16) * GPB);
            f.z[c] = 0x08080808u;
            if constexpr (ZEROS) f.z[c] = *(const typename Zeros<GPB>::type*)(g.zeros + (tile * 16 + l16) * GPB);
        }
    };
    const WidenF16 widen_f16;
    const WidenI8<ZEROS> widen_i8;
    floatx4 acc[T][TM];
#pragma unroll
    for (int c = 0; c < T; ++c)
#pragma unroll
        for (int i = 0; i < TM; ++i) acc[c][i] = floatx4{0, 0, 0, 0};
    const auto multiply = [&](const Codes& f, uint32_t kt) __attribute__((always_inline)) {
        constexpr int STEPS = 4 / GPB;                     // words of a group
        static_for<0, GPB>([&](auto qc) {
            constexpr int q = decltype(qc)::value;
            P_t part[T][TM], none = {0, 0, 0, 0};
            asm volatile("" : "+v"(none));                 // (one quad of zeros, not one for every product)
            float s[T];
            WidenF16::Zero zf[T];
            uint32_t zi[T];
#pragma unroll
            for (int c = 0; c < T; ++c) {
                if constexpr (GPB == 1) s[c] = (float)f.s[c]; else s[c] = (float)f.s[c][q];
                s[c] *= Factor<I8, ZEROS>::value;
                if (kt * kQ4TileCols + q * (kQ4TileCols / GPB) >= g.K) s[c] = 0.f;       // a group beyond the last column
                const uint32_t z = (f.z[c] >> (8 * q)) & 0xffu;
                zf[c] = WidenF16::zero(z);
                zi[c] = z * 0x01010101u;
            }
            // words taken together: two of an int8 group (64 columns), one otherwise
            constexpr int BY = I8 && STEPS > 1 ? 2 : 1;
            static_for<0, STEPS / BY>([&](auto jc) {
                constexpr int j = q * STEPS + decltype(jc)::value * BY;
                uintx4 x[TM];
#pragma unroll
                for (int i = 0; i < TM; ++i) {
                    x[i] = *(const uintx4*)(turn + (16 * i + held) * R::BYTES + R::slot((I8 ? j / 2 : j) * 4 + kg, held));
                    if constexpr (I8 && BY == 1 && j % 2) { x[i][0] = x[i][2]; x[i][1] = x[i][3]; }
                }
#pragma unroll
                for (int c = 0; c < T; ++c) {
                    if constexpr (!I8) {
                        const halfx8 wf = widen_f16(f.w[c][j], zf[c]);
#pragma unroll
                        for (int i = 0; i < TM; ++i)
                            part[c][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(halfx8, x[i]), wf, decltype(jc)::value == 0 ? none : part[c][i], 0, 0, 0);
                    } else if constexpr (BY == 1) {
                        const uintx2 wi = widen_i8(f.w[c][j], zi[c]);
#pragma unroll
                        for (int i = 0; i < TM; ++i)
                            part[c][i] = __builtin_amdgcn_mfma_i32_16x16x32_i8(__builtin_bit_cast(long, uintx2{x[i][0], x[i][1]}), __builtin_bit_cast(long, wi), none, 0, 0, 0);
                    } else {
                        const uintx2 w0 = widen_i8(f.w[c][j], zi[c]), w1 = widen_i8(f.w[c][j + 1], zi[c]);
                        const intx4 b = {(int)w0[0], (int)w0[1], (int)w1[0], (int)w1[1]};
#pragma unroll
                        for (int i = 0; i < TM; ++i)
                            part[c][i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(intx4, x[i]), b, decltype(jc)::value == 0 ? none : part[c][i], 0, 0, 0);
                    }
                }
            });
#pragma unroll
            for (int c = 0; c < T; ++c)
#pragma unroll
                for (int i = 0; i < TM; ++i) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[c][i][e] = __builtin_fmaf((float)part[c][i][e], s[c], acc[c][i][e]);
                    asm volatile("" : "+v"(acc[c][i]));    // (here and now: put off to where acc is next needed, the parts would live until then)
                }
        });
    };

    // codes for two steps, taking turns; X is asked for before them, since loads are waited for in their order
    Codes a, b;
    uint32_t kt = wave;
    const auto step = [&](const Codes& now, Codes& next) __attribute__((always_inline)) {
        turn_rows(kt);
        if constexpr (AHEAD_ALWAYS) {
            fetch_rows(kt + WAVES);
            fetch_codes(next, kt + WAVES < g.k_tiles ? kt + WAVES : kt);
        } else if (kt + WAVES < g.k_tiles) {
            fetch_codes(next, kt + WAVES);
            fetch_rows(kt + WAVES);
        }
        multiply(now, kt);
        kt += WAVES;
        return kt < g.k_tiles;
    };
    if (kt < g.k_tiles) {
        if constexpr (AHEAD_ALWAYS) fetch_rows(kt);
        fetch_codes(a, kt);
        if constexpr (!AHEAD_ALWAYS) fetch_rows(kt);
        while (step(a, b) && step(b, a)) {}
    }
    __syncthreads();
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

// ---- many rows -------------------------------------------------------------------------------------------------------
//
// A workgroup owns BM = 16 TM WM rows of X and BN = 16 TN WN columns of Y; a wavefront (wm, wn) of it 16 TM x 16 TN.  X goes
// through LDS, one column tile of W (128 of K) per stage, two stages; its global loads travel through registers, so that they
// may be unaligned and int8 can be put into the order of the codes on the way.  The codes need no LDS: a wavefront loads the
// pieces of its TN row tiles straight into the registers the matrix instruction reads them from, one stage ahead, and
// widens them there, once for all its TM tiles of X.
// Bound: the issue port that the vector pipe shares with the matrix pipe.  A SIMD takes a v_mfma of 16 cycles every 8 issue
// cycles at best and a vector instruction every 4; beside 96 of the former a column tile costs a wavefront of 128 x 48 about 235
// of the latter (9 a word to widen, 4 a tile and group to scale), 128 x 64 more registers than there are, 64 x 64 365.  So the
// large tile of 128 x 384 holds 8 wavefronts of 128 x 48: 4096 x 8192 x 8192 fp16 490 us (1122 TFLOP/s; 498 on a slower board, of
// that 8 % for a last round of three quarters, 7 % power: 460 with zeros in X), int8 319 (1724).  64 x 64 each: 510 and 346.
// Groups of 64 and 32 scale two and four times the sums: 3.7 and 5.9 vector instructions a product instead of 2.5, fp16 547 and
// 651 us.  The small tile shares what a column and group costs among four tiles of X: 1000 x 4096 x 8192 int8 in groups of 64 with
// zero points has 15.6 vector instructions a product (8 scale, 3.5 widen, the rest looks after scales and zero points), 82 us.
// Holding one of a SIMD's two wavefronts back by half a step, so that one widens while the other multiplies: no gain (498 -> 549,
// int8 329 -> 340).
template <bool I8, int GPB, bool ZEROS, int TM, int TN, int WM, int WN>
__global__ void __launch_bounds__(WM * WN * 64)
__attribute__((amdgpu_waves_per_eu(TM * TN >= 16 ? 2 : 3)))
gemm_q4_tiles_kernel(const GemmQ4Args g)
{
    constexpr int NT = WM * WN * 64, BM = 16 * TM * WM, BN = 16 * TN * WN;
    typedef XRows<I8> R;
    typedef typename std::conditional<I8, signed char, _Float16>::type X_t;
    constexpr int ROW = R::BYTES, CPR = R::CHUNKS, STAGE = BM * ROW, CH = STAGE / 16 / NT;
    constexpr int STEPS = 4 / GPB, GROUP = 128 / GPB;
    constexpr int EPI = WM * WN * 16 * 16 * TN * 4;
    static_assert(CH >= 1 && CH * NT * 16 == STAGE, "whole chunks per thread");
    __shared__ __attribute__((aligned(1024))) unsigned char lds[2 * STAGE > EPI ? 2 * STAGE : EPI];
    typedef typename Scales<GPB>::type S_t;

    const int t = threadIdx.x, lane = t & 63, l16 = lane & 15, kg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6), wm = wave / WN, wn = wave % WN;
    uint32_t tile_m, tile_n, z;
    {
        // every XCD a contiguous range of tiles, walked in groups of 8 tile rows (of 4: 4096 x 8192 x 8192 1.3 % slower)
        const uint32_t tiles = g.tiles_m * g.tiles_n;
        z = blockIdx.x / tiles;
        GemmArgs map;
        map.tiles_m = g.tiles_m; map.tiles_n = g.tiles_n; map.group_m = 8;
        block_to_tile(map, blockIdx.x % tiles, tiles, 0, tile_m, tile_n);
    }
    const uint32_t m0 = tile_m * BM, n0 = tile_n * BN;
    const uint32_t kt0 = z * g.split_tiles, kt1 = kt0 + g.split_tiles < g.k_tiles ? kt0 + g.split_tiles : g.k_tiles;

    // ---- X: chunk c of this thread is the 16 bytes `at` of row `row`
    const unsigned char* src[CH];
    uint32_t dst[CH];
    const int at = t % CPR;                                // (NT is a multiple of the chunks of a row)
    static_assert(NT % CPR == 0, "");
    const auto row_of = [&](int c) {
        const uint32_t m = m0 + t / CPR + c * (NT / CPR);
        return (const unsigned char*)g.X + (size_t)(m < g.M ? m : g.M - 1) * g.ldx * (I8 ? 1 : 2);       // rows behind the last one: never stored
    };
    // (Nothing is fetched under a condition: registers that a branch may leave as they were are copied every step.  The columns
    // of a part of a tile are fetched as they are put; what is fetched in their place is another tile's, or with no whole tile
    // the first codes.)
    const uint32_t whole = g.K / 128;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        src[c] = whole ? row_of(c) + at * 16 : g.codes;
        dst[c] = R::place(t / CPR + c * (NT / CPR), at);
    }
    uintx4 staged[CH];
    const auto fetch_x = [&](uint32_t kt) {
        const size_t from = (size_t)(kt < whole ? kt : whole ? whole - 1 : 0) * ROW;
#pragma unroll
        for (int c = 0; c < CH; ++c) __builtin_memcpy(&staged[c], src[c] + from, 16);
    };
    const auto put_x = [&](uint32_t kt, int stage) {
        if ((kt + 1) * kQ4TileCols <= g.K) {
#pragma unroll
            for (int c = 0; c < CH; ++c) R::put(lds + stage * STAGE, dst[c], staged[c]);
        } else {
#pragma unroll 1
            for (int c = 0; c < CH; ++c)
                R::put(lds + stage * STAGE, R::place(t / CPR + c * (NT / CPR), at), load_end((const X_t*)row_of(c), kt * 128 + at * (I8 ? 16 : 8), g.K));
        }
    };

    // ---- W
    size_t tile_at[TN];
#pragma unroll
    for (int c = 0; c < TN; ++c) {
        const uint32_t nt = n0 / 16 + wn * TN + c;
        tile_at[c] = (size_t)(nt < g.n_tiles ? nt : g.n_tiles - 1) * g.k_tiles;
    }
    uintx4 w[TN];
    S_t sv[TN];
    uint32_t zv[TN];
    const auto fetch_w = [&](uint32_t kt) {
#pragma unroll
        for (int c = 0; c < TN; ++c) {
            const size_t tile = tile_at[c] + kt;
            w[c] = *(const uintx4*)(g.codes + tile * kQ4TileBytes + lane * 16);
            sv[c] = *(const S_t*)(g.scales + (tile * 16 + l16) * GPB);
            zv[c] = 0x08080808u;
            if constexpr (ZEROS) zv[c] = *(const typename Zeros<GPB>::type*)(g.zeros + (tile * 16 + l16) * GPB);
        }
    };

    const WidenF16 widen_f16;
    const WidenI8<ZEROS> widen_i8;
    floatx4 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int c = 0; c < TN; ++c) acc[i][c] = floatx4{0, 0, 0, 0};

    const uint32_t frag_row = (wm * 16 * TM + l16) * ROW;
    // One group at a time: its codes widened, then (TM tiles of X) x (steps of the group), the fragment of X three steps ahead
    // on its way from LDS.  The sums of a tile are scaled behind the first product of the next one.  (The barriers to the
    // scheduler keep the widened codes of other groups, and more fragments than these, out of the registers.)
    typedef typename std::conditional<I8, intx4, floatx4>::type P_t;
    constexpr int XS = I8 && STEPS > 1 ? STEPS / 2 : STEPS, ALL = TM * XS, AHEAD = 3;    // products a tile and group, in all, fragments ahead
    halfx8 wf[I8 ? 1 : TN][STEPS];
    uintx2 wi[I8 ? TN : 1][STEPS];
    float s[TN];
    uintx4 wc[TN];
    S_t sc[TN];
    uint32_t zc[TN];
    const auto widen = [&](uint32_t kt, auto qc) __attribute__((always_inline)) {
        constexpr int q = decltype(qc)::value;
#pragma unroll
        for (int c = 0; c < TN; ++c) {
            if constexpr (GPB == 1) s[c] = (float)sc[c]; else s[c] = (float)sc[c][q];
            s[c] *= Factor<I8, ZEROS>::value;
            if (kt * 128 + q * GROUP >= g.K) s[c] = 0.f;             // a group beyond the last column
            const uint32_t zero = (zc[c] >> (8 * q)) & 0xffu;
#pragma unroll
            for (int j = 0; j < STEPS; ++j) {
                if constexpr (I8) wi[c][j] = widen_i8(wc[c][q * STEPS + j], zero * 0x01010101u);
                else wf[c][j] = widen_f16(wc[c][q * STEPS + j], WidenF16::zero(zero));
            }
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    const auto multiply = [&](const unsigned char* from, auto qc) __attribute__((always_inline)) {
        constexpr int q = decltype(qc)::value;
        P_t part[2][TN], none = {0, 0, 0, 0};
        asm volatile("" : "+v"(none));                     // (else every tile's and group's zeros are four registers of their own, kept across the loop)
        uintx4 x[AHEAD + 1];
        const auto read_x = [&](auto fc) {
            constexpr int f = decltype(fc)::value, i = f / XS, j = f % XS;
            if constexpr (f < ALL) {
                constexpr int chunk = I8 ? (STEPS == 1 ? q / 2 : q * XS + j) * 4 : (q * STEPS + j) * 4;
                x[f % (AHEAD + 1)] = *(const uintx4*)(from + i * 16 * ROW + R::slot(chunk + kg, l16));
            }
        };
        static_for<0, AHEAD>(read_x);
        const auto scale = [&](auto ic) {
            constexpr int i = decltype(ic)::value;
#pragma unroll
            for (int c = 0; c < TN; ++c) {
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][c][e] = __builtin_fmaf((float)part[i & 1][c][e], s[c], acc[i][c][e]);
                asm volatile("" : "+v"(acc[i][c]));        // (else these are moved to the loop's end, where acc is next needed, and every part lives until then)
            }
        };
        static_for<0, ALL>([&](auto fc) {
            constexpr int f = decltype(fc)::value, i = f / XS, j = f % XS;
            read_x(std::integral_constant<int, f + AHEAD>{});
            const uintx4 xv = x[f % (AHEAD + 1)];
#pragma unroll
            for (int c = 0; c < TN; ++c) {
                const P_t old = j == 0 ? none : part[i & 1][c];
                if constexpr (!I8) {
                    part[i & 1][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(halfx8, xv), wf[c][j], old, 0, 0, 0);
                } else if constexpr (STEPS == 1) {
                    const uintx2 xh = q % 2 ? uintx2{xv[2], xv[3]} : uintx2{xv[0], xv[1]};
                    part[i & 1][c] = __builtin_amdgcn_mfma_i32_16x16x32_i8(__builtin_bit_cast(long, xh), __builtin_bit_cast(long, wi[c][0]), old, 0, 0, 0);
                } else {
                    const intx4 b = {(int)wi[c][2 * j][0], (int)wi[c][2 * j][1], (int)wi[c][2 * j + 1][0], (int)wi[c][2 * j + 1][1]};
                    part[i & 1][c] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(intx4, xv), b, old, 0, 0, 0);
                }
            }
            if constexpr (j == 0 && i > 0) scale(std::integral_constant<int, i - 1>{});
            __builtin_amdgcn_sched_barrier(0);
        });
        scale(std::integral_constant<int, TM - 1>{});
        __builtin_amdgcn_sched_barrier(0);
    };
    const auto meet = [] { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };
    if (kt0 < kt1) {
        fetch_x(kt0);
        fetch_w(kt0);
        put_x(kt0, 0);
    }
    meet();
    for (uint32_t kt = kt0; kt < kt1; ++kt) {
        const unsigned char* from = lds + ((kt - kt0) & 1) * STAGE + frag_row;
        const bool more = kt + 1 < kt1;
        const uint32_t next = more ? kt + 1 : kt;
        fetch_x(next);
#pragma unroll
        for (int c = 0; c < TN; ++c) { wc[c] = w[c]; sc[c] = sv[c]; zc[c] = zv[c]; }
        if (GPB > 1) fetch_w(next);
        static_for<0, GPB>([&](auto qc) {
            widen(kt, qc);
            if (GPB == 1) fetch_w(next);
            multiply(from, qc);
        });
        if (more) put_x(kt + 1, (kt + 1 - kt0) & 1);
        meet();
    }

    // Epilogue: 16 rows at a time through a buffer of the wavefront's own, so that rows are stored 4 columns a lane
    float* const turn = (float*)lds + wave * (16 * 16 * TN);
    constexpr int QUADS = 4 * TN;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
#pragma unroll
        for (int c = 0; c < TN; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) turn[(4 * kg + e) * (16 * TN) + 16 * c + l16] = acc[i][c][e];
        wavefront_order();
#pragma unroll
        for (int p = 0; p < TN; ++p) {
            const int r = (p * 64 + lane) / QUADS;
            const uint32_t col = (p * 64 + lane) % QUADS * 4, m = m0 + wm * 16 * TM + 16 * i + r, n = n0 + wn * 16 * TN + col;
            const floatx4 v = *(const floatx4*)(turn + r * (16 * TN) + col);
            if (m < g.M && n < g.N) {
                if (g.splits > 1) {
                    float* out = g.partial + ((size_t)z * g.M + m) * g.partial_ld + n;       // (a whole piece: the pitch is a multiple of 4)
                    *(floatx4*)out = v;
                } else {
                    store_y4(g, m, n, v);
                }
            }
        }
        wavefront_order();
    }
}

// The ranges' sums, in their order, and the epilogue.
__global__ void __launch_bounds__(256) gemm_q4_join_kernel(const GemmQ4Args g)
{
    const uint32_t quads = g.partial_ld / 4;
    const uint64_t all = (uint64_t)quads * g.M;
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (uint64_t)gridDim.x * 256) {
        const uint32_t m = (uint32_t)(i / quads), n = (uint32_t)(i % quads) * 4;
        const float* from = g.partial + (size_t)m * g.partial_ld + n;
        const size_t step = (size_t)g.M * g.partial_ld;
        floatx4 v = *(const floatx4*)from;
        for (uint32_t z = 1; z < g.splits; ++z) {
            const floatx4 p = *(const floatx4*)(from + z * step);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] += p[e];
        }
        store_y4(g, m, n, v);
    }
}

namespace {

// Rows that one launch of a kernel of few rows takes: a grid has at most 65535 workgroups in y, a launch fewer than 2^32 threads.
// (Outputs of a few columns and millions of rows: 5000000 x 16 x 512 would have 78125.)
uint32_t rows_a_launch(uint32_t across, uint32_t tm, uint32_t waves)
{
    const uint32_t by_threads = 0xffffffffu / (waves * 64) / across;
    return (by_threads < 65535u ? by_threads : 65535u) * 16 * tm;
}

template <bool I8, int GPB, bool ZEROS, int TM, int T, int WAVES, int CH = (I8 ? 2 : 4) * TM> int launch_rows(const GemmQ4Args& args, hipStream_t stream)
{
    const uint32_t across = (args.n_tiles + T - 1) / T, most = rows_a_launch(across, TM, WAVES);
    const size_t y_bytes = args.y_f32 ? 4 : 2;
    for (uint64_t m0 = 0; m0 < args.M; m0 += most) {
        GemmQ4Args g = args;
        g.M = args.M - m0 < most ? (uint32_t)(args.M - m0) : most;
        g.X = (const char*)args.X + m0 * args.ldx * (I8 ? 1 : 2);
        if (args.x_scales) g.x_scales = args.x_scales + m0;
        if (args.C) g.C = (const char*)args.C + m0 * args.ldc * y_bytes;
        g.Y = (char*)args.Y + m0 * args.ldy * y_bytes;
        hipLaunchKernelGGL((gemm_q4_rows_kernel<I8, GPB, ZEROS, TM, T, WAVES, CH>), dim3(across, (g.M + 16 * TM - 1) / (16 * TM)), dim3(WAVES * 64), 0, stream, g);
        const hipError_t err = hipGetLastError();
        if (err != hipSuccess) return (int)err;
    }
    return 0;
}

template <bool I8, int GPB, bool ZEROS, int TM, int TN, int WM, int WN> int launch_tiles(const GemmQ4Args& args, hipStream_t stream)
{
    GemmQ4Args g = args;
    constexpr uint32_t BM = 16 * TM * WM, BN = 16 * TN * WN;
    g.tiles_m = (g.M + BM - 1) / BM;
    g.tiles_n = (g.N + BN - 1) / BN;
    hipLaunchKernelGGL((gemm_q4_tiles_kernel<I8, GPB, ZEROS, TM, TN, WM, WN>), dim3(g.tiles_m * g.tiles_n * g.splits), dim3(WM * WN * 64), 0, stream, g);
    if (g.splits > 1) {
        const uint64_t want = ((uint64_t)g.partial_ld / 4 * g.M + 255) / 256;
        hipLaunchKernelGGL(gemm_q4_join_kernel, dim3((unsigned)(want < 2048 ? want : 2048)), dim3(256), 0, stream, g);
    }
    return (int)hipGetLastError();
}

template <bool I8, int GPB, bool ZEROS> int launch_for(const GemmQ4Args& g, const GemmQ4Plan& p, hipStream_t stream)
{
    if (g.M <= (I8 ? 8 : 4)) {                             // (one load of X: fewer registers, less of the L1)
        switch (p.kernel) {
        case Q4_ROWS_16_NARROW: return launch_rows<I8, GPB, ZEROS, 1, 1, 16, 1>(g, stream);
        case Q4_ROWS_16:        return launch_rows<I8, GPB, ZEROS, 1, 2, 16, 1>(g, stream);
        default:                return launch_rows<I8, GPB, ZEROS, 1, 2, 8, 1>(g, stream);
        }
    }
    if constexpr (!I8)
        if (g.M <= 8) {                                    // (two: 7 x 5003 x 7001, whose rows are not aligned, 9.4 us with four, 7.7 so)
            switch (p.kernel) {
            case Q4_ROWS_16_NARROW: return launch_rows<I8, GPB, ZEROS, 1, 1, 16, 2>(g, stream);
            case Q4_ROWS_16:        return launch_rows<I8, GPB, ZEROS, 1, 2, 16, 2>(g, stream);
            default:                return launch_rows<I8, GPB, ZEROS, 1, 2, 8, 2>(g, stream);
            }
        }
    switch (p.kernel) {
    case Q4_ROWS_16_NARROW: return launch_rows<I8, GPB, ZEROS, 1, 1, 16>(g, stream);
    case Q4_ROWS_16:        return launch_rows<I8, GPB, ZEROS, 1, 2, 16>(g, stream);
    case Q4_ROWS_16_WIDE:   return launch_rows<I8, GPB, ZEROS, 1, 2, 8>(g, stream);
    case Q4_ROWS_32_NARROW: return launch_rows<I8, GPB, ZEROS, 2, 1, 8>(g, stream);
    case Q4_ROWS_32:        return launch_rows<I8, GPB, ZEROS, 2, 2, 8>(g, stream);
    case Q4_ROWS_64_NARROW: return launch_rows<I8, GPB, ZEROS, 4, 1, 8>(g, stream);
    case Q4_ROWS_64:        return launch_rows<I8, GPB, ZEROS, 4, 2, 8>(g, stream);
    case Q4_TILES_64x128:   return launch_tiles<I8, GPB, ZEROS, 4, 2, 1, 4>(g, stream);
    case Q4_TILES_64x256:   return launch_tiles<I8, GPB, ZEROS, 4, 4, 1, 4>(g, stream);
    default:                return launch_tiles<I8, GPB, ZEROS, 8, 3, 1, 8>(g, stream);
    }
}

template <bool I8, int GPB> int launch_as(const GemmQ4Args& g, const GemmQ4Plan& p, hipStream_t stream)
{
    return g.zeros ? launch_for<I8, GPB, true>(g, p, stream) : launch_for<I8, GPB, false>(g, p, stream);
}

}  // namespace

// Which kernel, and how many ranges K is cut into.
// Up to 16 rows the codes decide alone.  One row tile of W per workgroup where there are no more than 256 (a workgroup per CU:
// 1 x 4096 x 16384 7.5 us, with two 10.2), else two, which halves what X costs (16 x 8192 x 8192 with 16 wavefronts 9.2 us, with
// one 11.5; 7 x 5003 x 7001 7.7, with one 9.9); 16 wavefronts per workgroup while there are few of them (7 x 5003 x 7001 7.7 us, with
// 8 8.4), 8 from 256 on (1 x 65536 x 8192 in groups of 32 53 us, with 16 61; 1 x 11008 x 4096 int8 6.1, with 16 7.6; 16 x 8192 x 8192
// 8.7, with 16 9.2).
// Beyond, by the time that each is expected to take: the figures in the code, microseconds, from sweeps of 100 to 4096 rows against
// 1024 to 11000 columns.  (Zero points are left out of it: they add 3 instructions a word, and 1000 x 4096 x 8192 int8 in groups of
// 64 is expected to take 64 us and takes 82 with them.)  A kernel of few rows takes `step` per column tile of a wavefront and round of 256 workgroups; a tiled
// one `alone` per column tile with one workgroup on a CU, `full` with as many as it holds.  Ranges pay for storing and reading
// their sums (7 MB/us) and a second launch; groups smaller than 128 for more sums to scale.  fp16: 128 x 8192 x 8192 on tiles of
// 64 x 128 in 4 ranges 27.0 us, whole 55.0, few-rows kernel 37.9 (int8 22.8, 45.2, 25.0); 100 x 4096 x 4096 in 8 ranges 13.9, in 4
// 13.9, whole 29.6, few-rows kernel 19.3; 60 x 8192 x 4096 int8 on the few-rows kernel 9.2, tiles in 4 ranges 13.1; 2048 x 4096 x 4096:
// 64 x 256 tiles 67.9 us, 64 x 128 77.0, 128 x 384 83.1; 4096 x 8192 x 8192: 510, 562, 492 (int8 346, 375, 319).
GemmQ4Plan plan_gemm_q4(bool i8, uint32_t group, uint32_t M, uint32_t N, uint32_t K, size_t workspace_bytes)
{
    const uint32_t nt = (N + kQ4TileRows - 1) / kQ4TileRows, kt = (K + kQ4TileCols - 1) / kQ4TileCols;
    const bool narrow = nt <= 256;
    if (M <= 16) return {narrow ? Q4_ROWS_16_NARROW : nt < 512 ? Q4_ROWS_16 : Q4_ROWS_16_WIDE, 1, kt};
    GemmQ4Plan best = {Q4_TILES_64x256, 1, kt};
    if (kt == 0) return best;
    double best_us = 1e30;
    const auto consider = [&](int kernel, uint32_t splits, uint32_t len, double us) {
        if (us < best_us) { best_us = us; best = {kernel, splits, len}; }
    };
    {
        const bool half = M <= 32;
        const uint64_t wgs = (uint64_t)((M + 63) / 64) * (narrow ? nt : (nt + 1) / 2);
        const double step = half ? (i8 ? 0.7 : 1.1) : (i8 ? 1.5 : 2.1), rounds = wgs <= 256 ? 1.0 : (double)((wgs + 255) / 256);
        consider(half ? (narrow ? Q4_ROWS_32_NARROW : Q4_ROWS_32) : (narrow ? Q4_ROWS_64_NARROW : Q4_ROWS_64), 1, kt,
                 rounds * step * (narrow ? 0.67 : 1.0) * ((kt + 7) / 8) * (group == 32 ? 1.2 : 1.0));
    }
    struct Tile { int kernel; uint32_t rows, columns, per_cu; double alone, full; };
    const Tile tiles[3] = {{Q4_TILES_128x384, 128, 384, 1, i8 ? 1.65 : 2.4, i8 ? 1.71 : 2.6}, {Q4_TILES_64x256, 64, 256, 2, i8 ? 1.05 : 1.34, i8 ? 1.39 : 2.03},
                           {Q4_TILES_64x128, 64, 128, 2, i8 ? 0.71 : 0.86, i8 ? 0.80 : 1.15}};
    const double finer = group == 128 ? 1.0 : group == 64 ? (i8 ? 1.25 : 1.13) : (i8 ? 1.6 : 1.41);
    const size_t sums = (size_t)M * ((N + 3) / 4 * 4) * 4;
    for (const Tile& t : tiles) {
        const uint64_t wgs = (uint64_t)((M + t.rows - 1) / t.rows) * ((N + t.columns - 1) / t.columns);
        for (uint32_t want = 1; want <= 8; ++want) {
            const uint32_t len = (kt + want - 1) / want, splits = len ? (kt + len - 1) / len : 1;
            if (splits != want || (want > 1 && (len < 2 || splits * sums > workspace_bytes))) continue;
            // one workgroup a CU: whole rounds; two: they drift apart, and a part of a round is a part of the time
            const uint64_t all = wgs * splits;
            const double round = (double)all / 512.0;
            double us = len * finer;
            if (all <= 256) us *= t.alone;
            else if (t.per_cu == 1) us *= t.full * (double)((all + 255) / 256);
            else us *= round <= 1.0 ? t.alone + (t.full - t.alone) * (2.0 * round - 1.0) : t.full * round;
            if (splits > 1) us += 2.0 + (double)splits * sums * 2.0 / 7e6;
            consider(t.kernel, splits, len, us);
        }
    }
    return best;
}

size_t gemm_q4_workspace(bool i8, uint32_t group, uint32_t M, uint32_t N, uint32_t K)
{
    const GemmQ4Plan p = plan_gemm_q4(i8, group, M, N, K, ~(size_t)0);
    return p.splits > 1 ? (size_t)p.splits * M * ((N + 3) / 4 * 4) * 4 : 0;
}

uint32_t gemm_q4_rows_a_launch(int kernel, uint32_t M, uint32_t N)
{
    const uint32_t nt = (N + kQ4TileRows - 1) / kQ4TileRows;
    const bool narrow = kernel == Q4_ROWS_16_NARROW || kernel == Q4_ROWS_32_NARROW || kernel == Q4_ROWS_64_NARROW;
    const uint32_t tm = kernel <= Q4_ROWS_16_WIDE ? 1 : kernel <= Q4_ROWS_32 ? 2 : 4;
    return kernel >= Q4_TILES_64x128 ? M : rows_a_launch(narrow ? nt : (nt + 1) / 2, tm, kernel <= Q4_ROWS_16 ? 16 : 8);
}

bool gemm_q4_plan_ok(const GemmQ4Plan& p, uint32_t M, uint32_t N, uint32_t K, size_t workspace_bytes)
{
    const uint32_t kt = (K + kQ4TileCols - 1) / kQ4TileCols;
    if (p.kernel < 0 || p.kernel >= Q4_KERNEL_COUNT || p.splits == 0) return false;
    if ((M <= 16) != (p.kernel <= Q4_ROWS_16_WIDE)) return false;
    if (p.kernel < Q4_TILES_64x128 && M > 16 && (M <= 32) != (p.kernel <= Q4_ROWS_32)) return false;
    if (p.splits == 1) return p.split_tiles == kt;
    const size_t sums = (size_t)M * ((N + 3) / 4 * 4) * 4;
    return p.kernel >= Q4_TILES_64x128 && p.splits <= 8 && p.split_tiles >= 2 && (kt + p.split_tiles - 1) / p.split_tiles == p.splits &&
           p.splits * sums <= workspace_bytes;
}

int launch_gemm_q4(bool i8, uint32_t group, const GemmQ4Args& args, const GemmQ4Plan& p, void* workspace, hipStream_t stream)
{
    GemmQ4Args g = args;
    g.splits = p.splits;
    g.split_tiles = p.split_tiles;
    g.partial = (float*)workspace;
    g.partial_ld = (g.N + 3) / 4 * 4;
    switch (group) {
    case 128: return i8 ? launch_as<true, 1>(g, p, stream) : launch_as<false, 1>(g, p, stream);
    case 64:  return i8 ? launch_as<true, 2>(g, p, stream) : launch_as<false, 2>(g, p, stream);
    default:  return i8 ? launch_as<true, 4>(g, p, stream) : launch_as<false, 4>(g, p, stream);
    }
}

}  // namespace decx_hip
