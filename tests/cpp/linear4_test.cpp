// de::GPU_Matrix4, Quantize4, Dequantize4, Linear4 and RMSNorm as a user of DECX.h calls them.
//   linear4_test host   without a GPU: every call is refused and leaves its outputs as they were
//   linear4_test gpu    a layer of two products against sums in 64 bits, the refusals, objects that share storage
#include "DECX.h"

#include <cmath>
#include <cstring>
#include <iostream>
#include <string>
#include <vector>

static int g_failures = 0;
#define CHECK(cond) do { if (!(cond)) { ++g_failures; std::cerr << "FAILED line " << __LINE__ << ": " #cond "\n"; } } while (0)

static uint64_t g_seed = 12345;
static double uniform()                                   // [-1, 1)
{
    g_seed = g_seed * 6364136223846793005ull + 1442695040888963407ull;
    return (double)(int64_t)(g_seed >> 11) / (double)(1ll << 52) - 1.0;
}

template <typename T> static T as(double v);
template <> float as<float>(double v) { return (float)v; }
template <> de::Half as<de::Half>(double v) { return de::Float2Half((float)v); }
static double of(float v) { return v; }
static double of(de::Half v) { return de::Half2Float(v); }
static double of(signed char v) { return v; }

typedef std::vector<std::vector<double>> Rows;

template <typename T> static de::GPU_Matrix& upload(const Rows& v, de::_DATA_TYPES_FLAGS_ type)
{
    const uint32_t h = (uint32_t)v.size(), w = (uint32_t)v[0].size();
    de::Matrix& host = de::CreateMatrixRef(type, w, h);
    for (uint32_t r = 0; r < h; ++r) for (uint32_t c = 0; c < w; ++c) *host.ptr<T>(r, c) = as<T>(v[r][c]);
    de::GPU_Matrix& dev = de::CreateGPUMatrixRef(type, w, h);
    CHECK(de::Memcpy(host, dev, {0, 0}, {0, 0}, {(int)w, (int)h}, de::DECX_MEMCPY_H2D).error_type == 0);
    host.release();
    return dev;
}
template <typename T> static Rows download(de::GPU_Matrix& dev)
{
    const uint32_t h = dev.Height(), w = dev.Width();
    de::Matrix& host = de::CreateMatrixRef(dev.Type(), w, h);
    CHECK(de::Memcpy(host, dev, {0, 0}, {0, 0}, {(int)w, (int)h}, de::DECX_MEMCPY_D2H).error_type == 0);
    Rows v(h, std::vector<double>(w));
    for (uint32_t r = 0; r < h; ++r) for (uint32_t c = 0; c < w; ++c) v[r][c] = of(*host.ptr<T>(r, c));
    host.release();
    return v;
}
template <typename T> static de::GPU_Vector& upload(const std::vector<double>& v, de::_DATA_TYPES_FLAGS_ type)
{
    de::Vector& host = de::CreateVectorRef(type, v.size());
    for (size_t i = 0; i < v.size(); ++i) *host.ptr<T>(i) = as<T>(v[i]);
    de::GPU_Vector& dev = de::CreateGPUVectorRef(type, v.size());
    CHECK(de::Memcpy(host, dev, 0, 0, v.size(), de::DECX_MEMCPY_H2D).error_type == 0);
    host.release();
    return dev;
}
static std::vector<double> download(de::GPU_Vector& dev)
{
    de::Vector& host = de::CreateVectorRef(dev.Type(), dev.Len());
    CHECK(de::Memcpy(host, dev, 0, 0, dev.Len(), de::DECX_MEMCPY_D2H).error_type == 0);
    std::vector<double> v(dev.Len());
    for (size_t i = 0; i < v.size(); ++i) v[i] = *host.ptr<float>(i);
    host.release();
    return v;
}
static Rows random_rows(uint32_t h, uint32_t w, double scale)
{
    Rows v(h, std::vector<double>(w));
    for (auto& r : v) for (double& e : r) e = of(as<de::Half>(uniform() * scale));
    return v;
}

// |got - want| <= adds 2^-23 sum |x w| (fp32 sums in any order), and half a step of fp16 where the result is one
static void compare(const Rows& got, const Rows& x, const std::vector<double>* xs, const Rows& w, const Rows* c, double alpha, double beta, bool f16, int line)
{
    const size_t K = w[0].size();
    bool fine = got.size() == x.size() && got[0].size() == w.size();
    for (size_t m = 0; fine && m < x.size(); ++m)
        for (size_t n = 0; n < w.size(); ++n) {
            double sum = 0, mag = 0;
            for (size_t k = 0; k < K; ++k) {
                const double p = x[m][k] * (xs ? (*xs)[m] : 1.0) * w[n][k];
                sum += p; mag += std::fabs(p);
            }
            double tol = ((double)K / 32 + 128 + 64 + 2) * std::ldexp(mag, -23), y = sum;
            if (c) {
                const double add = beta * (*c)[c->size() == 1 ? 0 : m][n];
                y = alpha * sum + add;
                tol = std::fabs(alpha) * tol + std::ldexp(std::fabs(alpha * sum) + std::fabs(add) + std::fabs(alpha) * tol, -23);
            }
            tol += f16 ? std::ldexp(std::fabs(y) + tol, -11) + std::ldexp(1.0, -25) : std::ldexp(std::fabs(y), -24);
            if (!(std::fabs(got[m][n] - y) <= tol)) { fine = false; std::cerr << "row " << m << " column " << n << ": " << got[m][n] << " for " << y << " (" << tol << ")\n"; break; }
        }
    if (!fine) { ++g_failures; std::cerr << "FAILED comparison of line " << line << "\n"; }
}

static int host_checks()
{
    de::GPU_Matrix4& w = de::CreateGPUMatrix4Ref();
    CHECK(w.Width() == 0 && w.Height() == 0 && w.Group() == 0 && !w.HasZeros());
    de::GPU_Matrix4* p = de::CreateGPUMatrix4Ptr();
    p->SoftCopy(w);
    p->release();
    de::GPU_Matrix& a = de::CreateGPUMatrixRef();
    de::GPU_Matrix& b = de::CreateGPUMatrixRef();
    de::GPU_Vector& v = de::CreateGPUVectorRef();
    const int not_init = decx::DECX_FAIL_CUDA_not_init;
    CHECK(de::nn::cuda::Quantize4(a, w).error_type == not_init);
    CHECK(de::nn::cuda::Dequantize4(w, a).error_type == not_init);
    CHECK(de::nn::cuda::Linear4(a, w, b).error_type == not_init);
    CHECK(de::nn::cuda::Linear4(a, v, w, b).error_type == not_init);
    CHECK(de::nn::cuda::Linear4(a, w, b, b, de::Number(1.f), de::Number(1.f)).error_type == not_init);
    CHECK(de::nn::cuda::RMSNorm(a, v, b).error_type == not_init);
    CHECK(de::nn::cuda::RMSNorm(a, a, v, b, b, v).error_type == not_init);
    CHECK(a.Type() == de::_VOID_ && b.Width() == 0);
    return g_failures;
}

static void one_layer(uint32_t rows, uint32_t cols, uint32_t hidden, uint32_t group, bool zeros)
{
    std::cout << "layer " << rows << " " << cols << " " << hidden << " " << group << " " << zeros << std::endl;
    const Rows w1 = random_rows(hidden, cols, 0.05), w2 = random_rows(cols, hidden, 0.05);
    de::GPU_Matrix& d1 = upload<float>(w1, de::_FP32_);
    de::GPU_Matrix& d2 = upload<de::Half>(w2, de::_FP16_);
    de::GPU_Matrix4& q1 = de::CreateGPUMatrix4Ref();
    de::GPU_Matrix4& q2 = de::CreateGPUMatrix4Ref();
    CHECK(de::nn::cuda::Quantize4(d1, q1, group, zeros).error_type == 0);
    CHECK(de::nn::cuda::Quantize4(d2, q2).error_type == 0);
    CHECK(q1.Width() == cols && q1.Height() == hidden && q1.Group() == group && q1.HasZeros() == zeros && q2.Group() == 128 && !q2.HasZeros());
    de::GPU_Matrix& back = de::CreateGPUMatrixRef();
    CHECK(de::nn::cuda::Dequantize4(q1, back, de::_FP32_).error_type == 0 && back.Type() == de::_FP32_);
    const Rows v1 = download<float>(back);
    CHECK(de::nn::cuda::Dequantize4(q2, back, de::_FP32_).error_type == 0);
    const Rows v2 = download<float>(back);
    double worst = 0;
    for (uint32_t n = 0; n < hidden; ++n) for (uint32_t k = 0; k < cols; ++k) worst = std::max(worst, std::fabs(v1[n][k] - w1[n][k]));
    CHECK(worst <= 0.1 / (zeros ? 15 : 14) * 1.01);        // a step of a group that spans 2 x 0.05: half from rounding, half from a rounded zero point
    const Rows x = random_rows(rows, cols, 1.0), r = random_rows(rows, cols, 3.0), weight = random_rows(1, cols, 1.0);
    de::GPU_Matrix& dx = upload<de::Half>(x, de::_FP16_);
    de::GPU_Matrix& dr = upload<de::Half>(r, de::_FP16_);
    de::GPU_Vector& dw = upload<de::Half>(weight[0], de::_FP16_);
    de::GPU_Matrix& codes = de::CreateGPUMatrixRef();
    de::GPU_Vector& scales = de::CreateGPUVectorRef();
    CHECK(de::nn::cuda::RMSNorm(dx, dr, dw, dr, codes, scales).error_type == 0);            // the sum stays in the residual
    CHECK(codes.Type() == de::_UINT8_ && scales.Len() == rows);
    const Rows sum = download<de::Half>(dr), c = download<signed char>(codes);
    const std::vector<double> s = download(scales);
    for (uint32_t m = 0; m < rows; ++m) {
        double squares = 0, top = 0;
        for (uint32_t k = 0; k < cols; ++k) {
            const double h = of(as<de::Half>((float)x[m][k] + (float)r[m][k]));
            CHECK(sum[m][k] == h);
            squares += h * h;
            top = std::max(top, std::fabs(h * weight[0][k]));
        }
        for (uint32_t k = 0; k < cols; ++k) CHECK(c[m][k] == std::nearbyint(127 * sum[m][k] * weight[0][k] / top));
        const double want = top / 127 / std::sqrt(squares / cols + 1e-5f);
        CHECK(std::fabs(s[m] - want) <= (cols / 64.0 + 40) * std::ldexp(want, -24));
    }
    de::GPU_Matrix& hid = de::CreateGPUMatrixRef();
    CHECK(de::nn::cuda::Linear4(codes, scales, q1, hid).error_type == 0 && hid.Type() == de::_FP16_ && hid.Width() == hidden && hid.Height() == rows);
    const Rows h = download<de::Half>(hid);
    compare(h, c, &s, v1, nullptr, 1, 1, true, __LINE__);
    de::GPU_Matrix& f32 = de::CreateGPUMatrixRef();
    CHECK(de::nn::cuda::Linear4(hid, q2, f32, de::Fp16_Accurate_L1).error_type == 0 && f32.Type() == de::_FP32_);
    compare(download<float>(f32), h, nullptr, v2, nullptr, 1, 1, false, __LINE__);
    // a bias row, and the residual in place
    const Rows bias = random_rows(1, cols, 1.0);
    de::GPU_Matrix& db = upload<de::Half>(bias, de::_FP16_);
    de::GPU_Matrix& out = de::CreateGPUMatrixRef();
    CHECK(de::nn::cuda::Linear4(hid, q2, db, out, de::Number(0.5f), de::Number(2.f)).error_type == 0);
    compare(download<de::Half>(out), h, nullptr, v2, &bias, 0.5, 2, true, __LINE__);
    CHECK(de::nn::cuda::Linear4(hid, q2, dr, dr, de::Number(de::Float2Half(1.f)), de::Number(1.f)).error_type == 0);
    compare(download<de::Half>(dr), h, nullptr, v2, &sum, 1, 1, true, __LINE__);
    // plain norms, in place too
    CHECK(de::nn::cuda::RMSNorm(dx, dw, out).error_type == 0 && out.Type() == de::_FP16_);
    const Rows plain = download<de::Half>(out);
    CHECK(de::nn::cuda::RMSNorm(dx, dw, dx).error_type == 0);
    CHECK(download<de::Half>(dx) == plain);
    q1.release(); q2.release();
}

static int gpu_checks()
{
    de::InitCuda();
    one_layer(1, 200, 300, 64, false);
    one_layer(5, 130, 515, 32, true);
    one_layer(70, 384, 256, 128, true);
    // refusals leave the outputs as they were
    const int dims = decx::DECX_FAIL_DimsNotMatching, type = decx::DECX_FAIL_UNSUPPORTED_TYPE, param = decx::DECX_FAIL_INVALID_PARAM;
    de::GPU_Matrix& x = upload<de::Half>(random_rows(4, 64, 1), de::_FP16_);
    de::GPU_Matrix& x32 = upload<float>(random_rows(4, 64, 1), de::_FP32_);
    de::GPU_Matrix& w = upload<float>(random_rows(32, 64, 1), de::_FP32_);
    de::GPU_Matrix& other = upload<de::Half>(random_rows(4, 65, 1), de::_FP16_);
    de::GPU_Vector& v = upload<de::Half>(std::vector<double>(64, 1.0), de::_FP16_);
    de::GPU_Vector& v3 = upload<float>(std::vector<double>(3, 1.0), de::_FP32_);
    de::GPU_Matrix4& q = de::CreateGPUMatrix4Ref();
    de::GPU_Matrix& y = de::CreateGPUMatrixRef();
    CHECK(de::nn::cuda::Linear4(x, q, y).error_type == decx::DECX_FAIL_CLASS_NOT_INIT);
    CHECK(de::nn::cuda::Quantize4(w, q, 48).error_type == param && q.Width() == 0);
    CHECK(de::nn::cuda::Quantize4(w, q, 32).error_type == 0 && q.Width() == 64 && q.Height() == 32);
    CHECK(de::nn::cuda::Linear4(x32, q, y).error_type == type && de::nn::cuda::Linear4(other, q, y).error_type == dims);
    CHECK(de::nn::cuda::Linear4(x, v3, q, y).error_type == type && de::nn::cuda::Linear4(x, q, x).error_type == param);
    CHECK(de::nn::cuda::Linear4(x, q, other, y, de::Number(1.f), de::Number(1.f)).error_type == dims);
    CHECK(de::nn::cuda::Linear4(x, q, y, 3).error_type == param && y.Width() == 0);
    CHECK(de::nn::cuda::RMSNorm(x, v, y, -1.f).error_type == param && de::nn::cuda::RMSNorm(other, v, y).error_type == dims);
    CHECK(de::nn::cuda::RMSNorm(x32, v, y).error_type == decx::DECX_FAIL_TYPE_MOT_MATCH);
    CHECK(de::nn::cuda::RMSNorm(x, v, x, v3).error_type == param);          // codes over the rows they come from
    CHECK(y.Width() == 0 && x.Type() == de::_FP16_ && v3.Len() == 3);
    de::GPU_Matrix& row = upload<de::Half>(random_rows(1, 32, 1), de::_FP16_);
    CHECK(de::nn::cuda::Linear4(x, q, row, row, de::Number(1.f), de::Number(1.f)).error_type == param && row.Height() == 1);
    CHECK(de::nn::cuda::Linear4(x, q, row, y, de::Number(1.0), de::Number(1.f)).error_type == decx::DECX_FAIL_TYPE_MOT_MATCH);
    // an alias keeps its weights when the original is made anew or released
    de::GPU_Matrix4& alias = de::CreateGPUMatrix4Ref();
    alias.SoftCopy(q);
    CHECK(de::nn::cuda::Linear4(x, q, y).error_type == 0);
    const Rows before = download<de::Half>(y);
    CHECK(de::nn::cuda::Quantize4(upload<float>(random_rows(32, 64, 1), de::_FP32_), q, 64, true).error_type == 0);
    q.release();
    CHECK(alias.Group() == 32 && !alias.HasZeros() && de::nn::cuda::Linear4(x, alias, y).error_type == 0);
    CHECK(download<de::Half>(y) == before);
    return g_failures;
}

int main(int argc, char** argv)
{
    const std::string mode = argc > 1 ? argv[1] : "host";
    const int rc = mode == "gpu" ? gpu_checks() : host_checks();
    std::cout << (rc ? "failed" : "ok") << std::endl;
    return rc ? 1 : 0;
}
