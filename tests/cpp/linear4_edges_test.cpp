// de::nn::cuda::Linear4, Quantize4 and RMSNorm at the edges of what their objects may be (needs a GPU).
//   linear4_edges_test <name of a check>
#include "DECX.h"

#include <cmath>
#include <cstring>
#include <iostream>
#include <string>
#include <vector>

static int g_failures = 0;
#define CHECK(cond) do { if (!(cond)) { ++g_failures; std::cerr << "FAILED line " << __LINE__ << ": " #cond "\n"; } } while (0)

static uint64_t g_seed = 777;
static float uniform()                                    // [-1, 1), a multiple of 2^-7: exact in fp16
{
    g_seed = g_seed * 6364136223846793005ull + 1442695040888963407ull;
    return (float)((int)(g_seed >> 56) - 128) / 128.f;
}

template <typename T> static T as(float v);
template <> float as<float>(float v) { return v; }
template <> de::Half as<de::Half>(float v) { return de::Float2Half(v); }
static float of(float v) { return v; }
static float of(de::Half v) { return de::Half2Float(v); }
static float of(signed char v) { return v; }

typedef std::vector<float> Values;                        // row after row

template <typename T> static de::GPU_Matrix& upload(const Values& v, uint32_t w, uint32_t h, de::_DATA_TYPES_FLAGS_ type)
{
    de::Matrix& host = de::CreateMatrixRef(type, w, h);
    for (uint32_t r = 0; r < h; ++r) for (uint32_t c = 0; c < w; ++c) *host.ptr<T>(r, c) = as<T>(v[(size_t)r * w + c]);
    de::GPU_Matrix& dev = de::CreateGPUMatrixRef(type, w, h);
    CHECK(de::Memcpy(host, dev, {0, 0}, {0, 0}, {(int)w, (int)h}, de::DECX_MEMCPY_H2D).error_type == 0);
    host.release();
    return dev;
}
template <typename T> static Values download(de::GPU_Matrix& dev)
{
    const uint32_t h = dev.Height(), w = dev.Width();
    de::Matrix& host = de::CreateMatrixRef(dev.Type(), w, h);
    CHECK(de::Memcpy(host, dev, {0, 0}, {0, 0}, {(int)w, (int)h}, de::DECX_MEMCPY_D2H).error_type == 0);
    Values v((size_t)h * w);
    for (uint32_t r = 0; r < h; ++r) for (uint32_t c = 0; c < w; ++c) v[(size_t)r * w + c] = of(*host.ptr<T>(r, c));
    host.release();
    return v;
}
static de::GPU_Vector& upload(const Values& v)
{
    de::Vector& host = de::CreateVectorRef(de::_FP16_, v.size());
    for (size_t i = 0; i < v.size(); ++i) *host.ptr<de::Half>(i) = as<de::Half>(v[i]);
    de::GPU_Vector& dev = de::CreateGPUVectorRef(de::_FP16_, v.size());
    CHECK(de::Memcpy(host, dev, 0, 0, v.size(), de::DECX_MEMCPY_H2D).error_type == 0);
    host.release();
    return dev;
}
static Values random_values(size_t n)
{
    Values v(n);
    for (float& e : v) e = uniform();
    return v;
}

static const int kParam = decx::DECX_FAIL_INVALID_PARAM, kType = decx::DECX_FAIL_UNSUPPORTED_TYPE;

// sum and dst one object, fresh or not: dst is written last
static void dst_is_the_sum()
{
    const uint32_t w = 70, h = 5;
    de::GPU_Matrix& x = upload<de::Half>(random_values(w * h), w, h, de::_FP16_);
    de::GPU_Matrix& r = upload<de::Half>(random_values(w * h), w, h, de::_FP16_);
    de::GPU_Vector& weight = upload(random_values(w));
    de::GPU_Matrix& sum = de::CreateGPUMatrixRef();
    de::GPU_Matrix& y = de::CreateGPUMatrixRef();
    CHECK(de::nn::cuda::RMSNorm(x, r, weight, sum, y).error_type == 0);
    const Values want = download<de::Half>(y);
    de::GPU_Matrix& fresh = de::CreateGPUMatrixRef();
    CHECK(de::nn::cuda::RMSNorm(x, r, weight, fresh, fresh).error_type == 0);
    CHECK(fresh.Type() == de::_FP16_ && fresh.Width() == w && fresh.Height() == h && download<de::Half>(fresh) == want);
    de::GPU_Matrix& other = upload<float>(random_values(300), 30, 10, de::_FP32_);          // of another shape and type, with room and without
    CHECK(de::nn::cuda::RMSNorm(x, r, weight, other, other).error_type == 0 && download<de::Half>(other) == want);
    de::GPU_Matrix& small = upload<float>(random_values(2), 2, 1, de::_FP32_);
    de::GPU_Matrix& alias = de::CreateGPUMatrixRef();
    alias.SoftCopy(small);
    CHECK(de::nn::cuda::RMSNorm(x, r, weight, small, alias).error_type == 0 && download<de::Half>(alias) == want);
    // codes cannot lie where the sum does
    de::GPU_Matrix& none = de::CreateGPUMatrixRef();
    de::GPU_Vector& scales = de::CreateGPUVectorRef();
    CHECK(de::nn::cuda::RMSNorm(x, r, weight, none, none, scales).error_type == kParam && none.Width() == 0 && scales.Len() == 0);
    // in place of the residual, and of the source, as before
    CHECK(de::nn::cuda::RMSNorm(x, r, weight, r, r).error_type == 0 && download<de::Half>(r) == want);
}


// sizes that the entry points below refuse: found out before the outputs are made anew
static void sizes_that_are_refused()
{
    de::GPU_Matrix& tall = de::CreateGPUMatrixRef(de::_FP16_, 1, 1u << 30);
    de::GPU_Matrix4& q = de::CreateGPUMatrix4Ref();
    CHECK(de::nn::cuda::Quantize4(tall, q).error_type == kParam && q.Width() == 0 && q.Height() == 0);      // 2^26 tiles
    tall.release();
    de::GPU_Matrix& outputs = de::CreateGPUMatrixRef(de::_FP16_, 1, (1u << 25) + 1);
    CHECK(de::nn::cuda::Quantize4(outputs, q).error_type == 0 && q.Height() == (1u << 25) + 1);
    de::GPU_Matrix& x = upload<de::Half>(random_values(2), 1, 2, de::_FP16_);
    de::GPU_Matrix& y = de::CreateGPUMatrixRef();
    CHECK(de::nn::cuda::Linear4(x, q, y).error_type == kParam && y.Width() == 0 && y.Height() == 0 && y.Type() == de::_VOID_);
    q.release();
    outputs.release();
    de::GPU_Matrix& rows = de::CreateGPUMatrixRef(de::_FP16_, 1, 1u << 31);
    de::GPU_Vector& weight = upload(random_values(1));
    de::GPU_Vector& scales = de::CreateGPUVectorRef();
    CHECK(de::nn::cuda::RMSNorm(rows, weight, y).error_type == kParam && y.Width() == 0);
    CHECK(de::nn::cuda::RMSNorm(rows, weight, y, scales).error_type == kParam && y.Width() == 0 && scales.Len() == 0);
    rows.release();
}

// outputs that were given another type before: storage of smaller elements is not taken for one of larger
static void outputs_of_another_type()
{
    const uint32_t w = 64, h = 200;
    de::GPU_Matrix& x = upload<de::Half>(random_values(w * h), w, h, de::_FP16_);
    de::GPU_Vector& weight = upload(random_values(w));
    de::GPU_Matrix& y = de::CreateGPUMatrixRef();
    de::GPU_Matrix& codes = de::CreateGPUMatrixRef();
    de::GPU_Vector& scales = de::CreateGPUVectorRef();
    CHECK(de::nn::cuda::RMSNorm(x, weight, y).error_type == 0 && de::nn::cuda::RMSNorm(x, weight, codes, scales).error_type == 0);
    const Values want = download<de::Half>(y), want_codes = download<signed char>(codes);
    de::GPU_Matrix& narrow = de::CreateGPUMatrixRef(de::_UINT8_, w, h);
    narrow.Reinterpret(de::_FP16_);
    CHECK(de::nn::cuda::RMSNorm(x, weight, narrow).error_type == 0 && download<de::Half>(narrow) == want);
    de::GPU_Matrix& wide = de::CreateGPUMatrixRef(de::_FP32_, w, h);
    wide.Reinterpret(de::_UINT8_);
    de::GPU_Vector& halves = de::CreateGPUVectorRef(de::_FP16_, h);
    halves.Reinterpret(de::_FP32_);
    CHECK(de::nn::cuda::RMSNorm(x, weight, wide, halves).error_type == 0 && download<signed char>(wide) == want_codes);
    de::Vector& a = de::CreateVectorRef(de::_FP32_, h);
    de::Vector& b = de::CreateVectorRef(de::_FP32_, h);
    CHECK(de::Memcpy(a, scales, 0, 0, h, de::DECX_MEMCPY_D2H).error_type == 0 && de::Memcpy(b, halves, 0, 0, h, de::DECX_MEMCPY_D2H).error_type == 0);
    for (uint32_t i = 0; i < h; ++i) CHECK(*a.ptr<float>(i) == *b.ptr<float>(i));
}

// inputs that were given another type: of another size refused, of the same one taken for what they are
static void inputs_of_another_type()
{
    const uint32_t w = 64, h = 4, n = 32;
    const Values values = random_values(w * h);
    de::GPU_Matrix& x = upload<de::Half>(values, w, h, de::_FP16_);
    de::GPU_Matrix& weights = upload<float>(random_values(w * n), w, n, de::_FP32_);
    de::GPU_Vector& weight = upload(random_values(w));
    de::GPU_Matrix4& q = de::CreateGPUMatrix4Ref();
    de::GPU_Matrix& y = de::CreateGPUMatrixRef();
    de::GPU_Vector& scales = de::CreateGPUVectorRef(de::_FP32_, h);
    de::GPU_Matrix& codes = de::CreateGPUMatrixRef(de::_UINT8_, w, h);
    CHECK(de::nn::cuda::Quantize4(weights, q).error_type == 0);
    de::GPU_Matrix& b16 = upload<de::Half>(values, w, h, de::_FP16_);
    b16.Reinterpret(de::_FP32_);
    de::GPU_Matrix& b8 = de::CreateGPUMatrixRef(de::_UINT8_, w, h);
    b8.Reinterpret(de::_FP16_);
    de::GPU_Matrix& c16 = de::CreateGPUMatrixRef(de::_FP16_, n, h);
    c16.Reinterpret(de::_FP32_);
    de::GPU_Vector& v16 = de::CreateGPUVectorRef(de::_FP16_, h);
    v16.Reinterpret(de::_FP32_);
    de::GPU_Vector& w8 = de::CreateGPUVectorRef(de::_UINT8_, w);
    w8.Reinterpret(de::_FP16_);
    CHECK(de::nn::cuda::Linear4(b8, q, y).error_type == kType);
    de::GPU_Matrix& alias = de::CreateGPUMatrixRef();
    alias.SoftCopy(b8);
    CHECK(de::nn::cuda::Linear4(alias, q, y).error_type == kType && de::nn::cuda::RMSNorm(alias, weight, y).error_type == kType);
    CHECK(de::nn::cuda::Linear4(x, q, c16, y, de::Number(1.f), de::Number(1.f)).error_type == kType);
    CHECK(de::nn::cuda::Linear4(codes, v16, q, y).error_type == kType);
    CHECK(de::nn::cuda::RMSNorm(b8, weight, y).error_type == kType && de::nn::cuda::RMSNorm(x, w8, y).error_type == kType);
    CHECK(de::nn::cuda::RMSNorm(x, b8, weight, y, codes).error_type == kType && codes.Type() == de::_UINT8_);
    de::GPU_Matrix4& none = de::CreateGPUMatrix4Ref();
    CHECK(de::nn::cuda::Quantize4(b16, none).error_type == kType && none.Width() == 0 && y.Width() == 0);
    CHECK(de::nn::cuda::Linear4(codes, scales, q, y).error_type == 0);
    de::GPU_Matrix& f32 = upload<float>(values, w, h, de::_FP32_);
    de::GPU_Matrix4& q1 = de::CreateGPUMatrix4Ref();
    de::GPU_Matrix4& q2 = de::CreateGPUMatrix4Ref();
    CHECK(de::nn::cuda::Quantize4(f32, q1).error_type == 0);
    f32.Reinterpret(de::_INT32_);
    f32.Reinterpret(de::_FP32_);
    CHECK(de::nn::cuda::Quantize4(f32, q2).error_type == 0);
    de::GPU_Matrix& v1 = de::CreateGPUMatrixRef();
    de::GPU_Matrix& v2 = de::CreateGPUMatrixRef();
    CHECK(de::nn::cuda::Dequantize4(q1, v1).error_type == 0 && de::nn::cuda::Dequantize4(q2, v2).error_type == 0);
    CHECK(download<de::Half>(v1) == download<de::Half>(v2));
}


int main(int argc, char** argv)
{
    const std::string name = argc > 1 ? argv[1] : "";
    de::InitCuda();
    if (name == "dst_is_the_sum") dst_is_the_sum();
    else if (name == "sizes_that_are_refused") sizes_that_are_refused();
    else if (name == "outputs_of_another_type") outputs_of_another_type();
    else if (name == "inputs_of_another_type") inputs_of_another_type();
    else { std::cerr << "no such check\n"; return 2; }
    std::cout << (g_failures ? "failed" : "ok") << std::endl;
    return g_failures ? 1 : 0;
}
