// Root-mean-square norm of rows, with the residual's addition in front and 8 bits behind:
//
//   h = x + residual (rounded to the rows' type, kept if asked for),  rho = 1 / sqrt(mean(h^2) + eps),  y = h * weight * rho
//   8 bits: top = max |h * weight| over the row,  code = rint(127 * h * weight / top),  scale = top * rho / 127
//
// rho cancels out of the codes, so they depend on h * weight alone: exact in fp32 for fp16 rows, in 64 bits for fp32 rows.  A
// quotient next to a half is decided by exact products, so no code depends on how one was rounded.
// Sums of squares are kept in fp32 for fp16 rows (a row cannot overflow it; of rows that are read twice only those of 8 elements and
// what a workgroup's threads end with) and in 64 bits for fp32 rows (they could overflow).
// Bound: HBM.  A workgroup owns a row and holds h in registers between the two passes over it; rows too long for that are
// read a second time (from the kept sum where there is one).  4096 x 8192 fp16 with residual, sum and 8 bits out: 45.9 us, 5.1 TB/s
// of 7 bytes an element (the calibration copy: 5.7); 777 x 5001 fp32 7.9 us; a single row of 4096 2.6 us, where a kernel with next
// to nothing to do takes 1.8.
#include "gemm_q4.hpp"

namespace decx_hip {

namespace {

typedef halfx8 halfx8_u __attribute__((aligned(2)));
typedef floatx4 floatx4_u __attribute__((aligned(4)));

// fp16 rows: 8 elements per 16 bytes, arithmetic in fp32.  fp32 rows: 4, in 64 bits.
template <typename T> struct Row;
template <> struct Row<_Float16> {
    static constexpr int n = 8;
    typedef halfx8 vec;
    typedef halfx8_u vec_u;
    typedef float wide;
    typedef uint32_t bits;
    static constexpr bits abs_mask = 0x7fffffffu, inf = 0x7f800000u;
};
template <> struct Row<float> {
    static constexpr int n = 4;
    typedef floatx4 vec;
    typedef floatx4_u vec_u;
    typedef double wide;
    typedef uint64_t bits;
    static constexpr bits abs_mask = 0x7fffffffffffffffull, inf = 0x7ff0000000000000ull;
};

template <typename T> __device__ __forceinline__ typename Row<T>::vec load_chunk(const T* row, uint32_t k, uint32_t cols)
{
    constexpr int n = Row<T>::n;
    if (k + n <= cols) return *(const typename Row<T>::vec_u*)(row + k);
    typename Row<T>::vec v;
#pragma unroll
    for (int e = 0; e < n; ++e) v[e] = k + e < cols ? row[k + e] : T(0);
    return v;
}
template <typename T> __device__ __forceinline__ void store_chunk(T* row, uint32_t k, uint32_t cols, const typename Row<T>::vec& v)
{
    constexpr int n = Row<T>::n;
    if (k + n <= cols) {
        *(typename Row<T>::vec_u*)(row + k) = v;
    } else {
#pragma unroll
        for (int e = 0; e < n; ++e) if (k + e < cols) row[k + e] = v[e];
    }
}

__device__ __forceinline__ uint32_t max_of(uint32_t a, uint32_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint64_t max_of(uint64_t a, uint64_t b) { return a > b ? a : b; }

// rint(127 t / top) by comparison with the half top (m + 1/2) next to the quotient, m = floor(v), v the quotient in fp32.  t and
// top are products of two elements: of fp16 ones 22 bits, and both sides are exact in 64 bits; of fp32 ones 48 bits, the sides take
// up to 56, and what each lost is compared behind them (the fma gives it exactly, and so is the difference of two such ends; the
// sides' own difference is exact next to a half, elsewhere larger than what they lost).
template <bool ENDS> __device__ __forceinline__ float rint_exactly(double t, double top, float v)
{
#pragma clang fp contract(off)                             // (the difference is that of the rounded sides)
    const float m = __builtin_floorf(v), even = 2.f * __builtin_rintf(0.5f * m + 0.25f);      // of m and m + 1 the even one
    const double left = 127.0 * t, half = top * (double)(m + 0.5f);
    double above = left - half;
    if constexpr (ENDS) above += __builtin_fma(127.0, t, -left) - __builtin_fma(top, (double)(m + 0.5f), -half);
    return above > 0 ? m + 1.f : (above < 0 ? m : even);
}

}  // namespace

// NT threads per row, CHUNKS 16-byte pieces of the row per thread (0: as many as it takes, read twice).
template <typename T, bool Q8, int NT, int CHUNKS>
__global__ void __launch_bounds__(NT)
rmsnorm_kernel(const RmsNormArgs g)
{
    typedef Row<T> R;
    typedef typename R::wide wide;
    typedef typename R::bits bits;
    constexpr int n = R::n, WAVES = NT / 64;
    const int t = threadIdx.x;
    const size_t r = blockIdx.x;
    const T* x = (const T*)g.x + r * g.ldx;
    const T* residual = g.residual ? (const T*)g.residual + r * g.ldr : nullptr;
    T* sum = g.sum ? (T*)g.sum + r * g.lds : nullptr;
    const T* weight = (const T*)g.weight;

    const auto add = [&](uint32_t k) {
        typename R::vec h = load_chunk(x, k, g.cols);
        if (residual) h += load_chunk(residual, k, g.cols);        // (packed fp16: rounded as a sum in fp32 rounded to fp16 is)
        return h;
    };
    wide squares = 0;
    bits top = 0;
    const auto gather = [&](const typename R::vec& h, const typename R::vec& w) {
#pragma unroll
        for (int e = 0; e < n; ++e) {
            const wide v = (wide)h[e];
            squares += v * v;
            if (Q8) top = max_of(top, __builtin_bit_cast(bits, v * (wide)w[e]) & R::abs_mask);
        }
    };
    typename R::vec held[CHUNKS > 0 ? CHUNKS : 1], w[CHUNKS > 0 ? CHUNKS : 1];
    if constexpr (CHUNKS > 0) {
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const uint32_t k = (uint32_t)(t + c * NT) * n;
            if (k < g.cols) {
                held[c] = add(k);
                w[c] = load_chunk(weight, k, g.cols);
            }
        }
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const uint32_t k = (uint32_t)(t + c * NT) * n;
            if (k < g.cols) {
                if (sum) store_chunk(sum, k, g.cols, held[c]);
                gather(held[c], w[c]);
            }
        }
    } else {
        double pieces = 0;                                 // (a thread adds as many as the row is long: its sum is kept in 64 bits)
        for (uint32_t k = (uint32_t)t * n; k < g.cols; k += NT * n) {
            const typename R::vec h = add(k);
            if (sum) store_chunk(sum, k, g.cols, h);
            squares = 0;
            gather(h, load_chunk(weight, k, g.cols));
            pieces += (double)squares;
        }
        squares = (wide)pieces;
    }
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) {
        squares += __shfl_xor(squares, off, 64);
        if (Q8) top = max_of(top, (bits)__shfl_xor((unsigned long long)top, off, 64));
    }
    if constexpr (WAVES > 1) {
        __shared__ wide all_squares[WAVES];
        __shared__ bits all_tops[WAVES];
        if ((t & 63) == 0) { all_squares[t >> 6] = squares; all_tops[t >> 6] = top; }
        __syncthreads();
        squares = 0; top = 0;
#pragma unroll
        for (int i = 0; i < WAVES; ++i) { squares += all_squares[i]; top = max_of(top, all_tops[i]); }
    }
    const wide mean = squares / (wide)g.cols + (wide)g.eps;
    wide rho;
    if constexpr (sizeof(wide) == 4) rho = 1.f / __builtin_sqrtf(mean); else rho = 1.0 / __builtin_sqrt(mean);
    const wide most = __builtin_bit_cast(wide, top);
    const bool finite = top < R::inf, some = top != 0 && finite;
    const wide inverse = some ? (wide)127 / most : (wide)0;
    if (Q8 && t == 0) g.y_scales[r] = some ? (float)(most * rho / (wide)127) : finite ? 0.f : __builtin_nanf("");

    const auto put = [&](uint32_t k, const typename R::vec& h, const typename R::vec& wv) {
        if constexpr (Q8) {
            // v is off by less than 127 * 2^-22; only where that is enough to cross a half is the exact form asked
            uint32_t word[2] = {0, 0};
            float v[n], c[n], near = 1.f;
#pragma unroll
            for (int e = 0; e < n; ++e) {
                v[e] = (float)((wide)h[e] * (wide)wv[e] * inverse);
                c[e] = __builtin_rintf(v[e]);
                near = __builtin_fminf(near, __builtin_fabsf(__builtin_fabsf(v[e] - c[e]) - 0.5f));
            }
            if (near < 4e-5f) {
#pragma unroll
                for (int e = 0; e < n; ++e) c[e] = rint_exactly<sizeof(T) == 4>((double)((wide)h[e] * (wide)wv[e]), (double)most, v[e]);
            }
#pragma unroll
            for (int e = 0; e < n; ++e) word[e / 4] |= ((uint32_t)(int)c[e] & 0xffu) << (8 * (e % 4));
            if (!some) word[0] = word[1] = 0;              // (a row of zeros, or one that meets what is not finite)
            unsigned char* out = (unsigned char*)g.y + r * g.ldy + k;
            if (k + n <= g.cols) {
                __builtin_memcpy(out, word, n);
            } else {
#pragma unroll
                for (int e = 0; e < n; ++e) if (k + e < g.cols) out[e] = (unsigned char)(word[e / 4] >> (8 * (e % 4)));
            }
        } else {
            typename R::vec y;
#pragma unroll
            for (int e = 0; e < n; ++e) y[e] = (T)((wide)h[e] * (wide)wv[e] * rho);
            store_chunk((T*)g.y + r * g.ldy, k, g.cols, y);
        }
    };
    if constexpr (CHUNKS > 0) {
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const uint32_t k = (uint32_t)(t + c * NT) * n;
            if (k < g.cols) put(k, held[c], w[c]);
        }
    } else {
        for (uint32_t k = (uint32_t)t * n; k < g.cols; k += NT * n)
            put(k, sum ? load_chunk((const T*)sum, k, g.cols) : add(k), load_chunk(weight, k, g.cols));
    }
}

namespace {

template <typename T, bool Q8> void launch_as(const RmsNormArgs& g, hipStream_t stream)
{
    const uint32_t chunks = (g.cols + Row<T>::n - 1) / Row<T>::n;
    const auto go = [&](auto nt, auto per) {
        constexpr int NT = decltype(nt)::value, CHUNKS = decltype(per)::value;
        hipLaunchKernelGGL((rmsnorm_kernel<T, Q8, NT, CHUNKS>), dim3(g.rows), dim3(NT), 0, stream, g);
    };
    // A thread per 16 bytes of an fp16 row while a workgroup has that many (4096 rows of 8192: 46.0 us, with two, four or eight
    // pieces a thread 48.5, 52.6, 58.5).  fp32 rows cost twice the arithmetic a byte: two pieces (4096 x 4096: 45.4 us, with
    // one 48.3), four where two would take 1024 threads (777 x 5001: 8.0 us against 9.7).  From 4096 pieces on (64 KB) the row
    // is read twice: 800 x 40000 fp16 63.9 us (63.7 with sums in fp32), held eight pieces a thread 64.7.
    using std::integral_constant;
    if (chunks <= 64) go(integral_constant<int, 64>{}, integral_constant<int, 1>{});
    else if (chunks <= 256) go(integral_constant<int, 256>{}, integral_constant<int, 1>{});
    else if (chunks <= 2048) {
        constexpr bool F32 = sizeof(T) == 4;
        if (chunks <= 1024) go(integral_constant<int, F32 ? 512 : 1024>{}, integral_constant<int, F32 ? 2 : 1>{});
        else go(integral_constant<int, F32 ? 512 : 1024>{}, integral_constant<int, F32 ? 4 : 2>{});
    }
    else if (chunks <= 4096) go(integral_constant<int, 1024>{}, integral_constant<int, 4>{});
    else go(integral_constant<int, 1024>{}, integral_constant<int, 0>{});
}

}  // namespace

int launch_rmsnorm(bool f16, const RmsNormArgs& args, hipStream_t stream)
{
    constexpr uint32_t MOST = 1u << 21;                    // rows a launch (it has fewer than 2^32 threads)
    const size_t e = f16 ? 2 : 4;
    for (uint64_t r0 = 0; r0 < args.rows; r0 += MOST) {
        RmsNormArgs g = args;
        g.rows = args.rows - r0 < MOST ? (uint32_t)(args.rows - r0) : MOST;
        g.x = (const char*)args.x + r0 * args.ldx * e;
        if (args.residual) g.residual = (const char*)args.residual + r0 * args.ldr * e;
        if (args.sum) g.sum = (char*)args.sum + r0 * args.lds * e;
        g.y = (char*)args.y + r0 * args.ldy * (args.y_scales ? 1 : e);
        if (args.y_scales) g.y_scales = args.y_scales + r0;
        if (f16) { if (g.y_scales) launch_as<_Float16, true>(g, stream); else launch_as<_Float16, false>(g, stream); }
        else     { if (g.y_scales) launch_as<float, true>(g, stream);    else launch_as<float, false>(g, stream); }
        const hipError_t err = hipGetLastError();
        if (err != hipSuccess) return (int)err;
    }
    return 0;
}

}  // namespace decx_hip
