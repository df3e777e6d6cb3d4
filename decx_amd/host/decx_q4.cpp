// Linear layers with weights in 4 bits, and the root-mean-square norm in front of them: the host side of
// de::GPU_Matrix4, de::nn::cuda::Quantize4 / Dequantize4 / Linear4 / RMSNorm, on the C ABI of decx_hip.h.
#include "decx_internal.hpp"

namespace decx {

class _GPU_Matrix4 : public de::GPU_Matrix4 {
    uint32_t _width = 0, _height = 0, _group = 0;
    std::shared_ptr<DeviceBlock> _codes, _scales, _zeros;

public:
    virtual uint Width() const { return _width; }
    virtual uint Height() const { return _height; }
    virtual uint Group() const { return _group; }
    virtual bool HasZeros() const { return _zeros != nullptr; }
    virtual void release() { _codes.reset(); _scales.reset(); _zeros.reset(); _width = _height = _group = 0; }
    virtual de::GPU_Matrix4& SoftCopy(de::GPU_Matrix4& src)
    {
        const _GPU_Matrix4& s = dynamic_cast<_GPU_Matrix4&>(src);
        if (this != &s) *this = s;
        return *this;
    }
    virtual ~_GPU_Matrix4() {}

    bool is_init() const { return _codes && _codes->ptr && _scales && _scales->ptr; }
    void* codes() const { return _codes->ptr; }
    uint16_t* scales() const { return (uint16_t*)_scales->ptr; }
    uint8_t* zeros() const { return _zeros ? (uint8_t*)_zeros->ptr : nullptr; }
    // storage of its own for a matrix of that shape (aliases keep what they had); false when the device has no room
    bool re_construct(uint32_t width, uint32_t height, uint32_t group, bool zeros)
    {
        const size_t count = decx_hip_q4_scales_count(height, width, group);
        const auto make = [](size_t bytes) {
            auto block = std::make_shared<DeviceBlock>();
            block->bytes = bytes;
            if (decx_hip_malloc(&block->ptr, bytes) != DECX_HIP_OK) { block->ptr = nullptr; block.reset(); }
            return block;
        };
        std::shared_ptr<DeviceBlock> c = make(decx_hip_q4_codes_bytes(height, width)), s = make(count * 2), z;
        if (zeros) z = make(count);
        if (!c || !s || (zeros && !z)) return false;
        _codes = c; _scales = s; _zeros = z;
        _width = width; _height = height; _group = group;
        return true;
    }
};

}  // namespace decx

namespace {

const char* const kCudaNotInit     = "error: CUDA should be initialized first";
const char* const kTypeNotMatch    = "error: The types of the two objects are not equal";
const char* const kDevAllocFail    = "error: Fail to allocate memory on device";
const char* const kClassNotInit    = "error: The class is not initialized";
const char* const kUnsupportedType = "error: The data type of the input onject is not supported";
const char* const kInvalidParam    = "error: The parameter(s) is(are) invalid";

de::DH failed(int code, const char* text)
{
    de::DH handle;
    decx::err::set(&handle, code, text);
    return handle;
}

// the ranges' sums of Linear4, kept between calls; grow-only, guarded by the module mutex
decx::DeviceBlock* workspace(size_t need)
{
    static std::shared_ptr<decx::DeviceBlock> kept;
    if (need == 0) return nullptr;
    if (!kept || kept->bytes < need) {
        auto block = std::make_shared<decx::DeviceBlock>();
        block->bytes = need;
        if (decx_hip_malloc(&block->ptr, need) != DECX_HIP_OK) { block->ptr = nullptr; return nullptr; }     // (the product does without)
        kept = block;
    }
    return kept.get();
}

// An input that was given another type (Reinterpret) keeps its pitch and storage: only elements of the same size are still there.
bool whole(const decx::_GPU_Matrix* m) { return !m || decx::element_size(m->Type()) == (uint32_t)m->get_layout()._single_element_size; }
bool whole(const decx::_GPU_Vector* v) { return !v || decx::element_size(v->Type()) == v->element_bytes(); }

float scalar_of(const de::Number& n) { return n.Type() == de::_FP16_ ? de::Half2Float(n.get_data_ref<de::Half>()) : n.get_data_ref<float>(); }

de::DH linear(de::GPU_Matrix& src, de::GPU_Vector* src_scales, de::GPU_Matrix4& weights, de::GPU_Matrix* C, de::GPU_Matrix& dst,
              const de::Number* alpha, const de::Number* beta, uint32_t accu)
{
    de::DH handle; decx::err::success(&handle);
    decx::_GPU_Matrix* x = dynamic_cast<decx::_GPU_Matrix*>(&src);
    decx::_GPU_Vector* xs = dynamic_cast<decx::_GPU_Vector*>(src_scales);
    decx::_GPU_Matrix4* w = dynamic_cast<decx::_GPU_Matrix4*>(&weights);
    decx::_GPU_Matrix* c = dynamic_cast<decx::_GPU_Matrix*>(C);
    decx::_GPU_Matrix* y = dynamic_cast<decx::_GPU_Matrix*>(&dst);
    if (!decx::gpu_ready()) return failed(decx::DECX_FAIL_CUDA_not_init, kCudaNotInit);
    if (!x || !w || !y || !x->is_init() || !w->is_init() || (src_scales && (!xs || !xs->is_init())) || (C && (!c || !c->is_init())))
        return failed(decx::DECX_FAIL_CLASS_NOT_INIT, kClassNotInit);
    if (x->Type() != (xs ? de::_UINT8_ : de::_FP16_) || (xs && xs->Type() != de::_FP32_) || (c && c->Type() != de::_FP16_ && c->Type() != de::_FP32_) || !whole(x) || !whole(xs) ||
        !whole(c))
        return failed(decx::DECX_FAIL_UNSUPPORTED_TYPE, kUnsupportedType);
    if (accu > de::Fp16_Accurate_L3) return failed(decx::DECX_FAIL_INVALID_PARAM, kInvalidParam);
    if (x->Width() != w->Width())
        return failed(decx::DECX_FAIL_DimsNotMatching, "The width of the source and of the weights must be identical");
    if (xs && xs->Len() != x->Height())
        return failed(decx::DECX_FAIL_DimsNotMatching, "There must be one scale for every row of the source");
    if (c && (c->Width() != w->Height() || (c->Height() != x->Height() && c->Height() != 1)))
        return failed(decx::DECX_FAIL_DimsNotMatching, "The matrix C must be of the result's size, or a single row of it");
    for (const de::Number* n : {alpha, beta})
        if (n && n->Type() != de::_FP32_ && n->Type() != c->Type())
            return failed(decx::DECX_FAIL_TYPE_MOT_MATCH, "The input scalar alpha and beta must be fp32 or match the type of C");
    // dst must not write over what is still read: its storage is the source's, or that of a row that all rows add
    if (y->is_init() && (y->data() == x->data() || (c && y->data() == c->data() && (c->Height() != x->Height() || y->Pitch() != c->Pitch() || y->Type() != c->Type()))))
        return failed(decx::DECX_FAIL_INVALID_PARAM, kInvalidParam);
    if (!decx_hip_gemm_q4_fits(x->Height(), w->Height(), w->Width(), w->Group())) return failed(decx::DECX_FAIL_INVALID_PARAM, kInvalidParam);
    const bool f32 = c ? c->Type() == de::_FP32_ : accu == de::Fp16_Accurate_L1;

    std::lock_guard<std::mutex> guard(decx::module_mutex());
    const uint32_t ldc = c ? (c->Height() == x->Height() ? c->Pitch() : 0) : 0;
    const void* c_ptr = c ? c->data() : nullptr;
    const uint32_t rows = x->Height();
    if (!y->re_construct(f32 ? de::_FP32_ : de::_FP16_, w->Height(), rows)) return *de::GetLastError();
    void* S = decx::module_stream();
    decx::DeviceBlock* ws = workspace(decx_hip_gemm_q4_workspace(xs ? 1 : 0, rows, w->Height(), w->Width(), w->Group()));
    const float a = alpha ? scalar_of(*alpha) : 1.f, b = beta ? scalar_of(*beta) : 1.f;
    int rc;
    if (xs)
        rc = decx_hip_gemm_q4_i8((const int8_t*)x->data(), (const float*)xs->data(), w->codes(), w->scales(), w->zeros(), c_ptr, y->data(), rows,
                                 w->Height(), w->Width(), w->Group(), x->Pitch(), ldc, y->Pitch(), a, b, f32, ws ? ws->ptr : nullptr,
                                 ws ? ws->bytes : 0, S);
    else
        rc = decx_hip_gemm_q4_f16((const uint16_t*)x->data(), w->codes(), w->scales(), w->zeros(), c_ptr, y->data(), rows, w->Height(),
                                  w->Width(), w->Group(), x->Pitch(), ldc, y->Pitch(), a, b, f32, ws ? ws->ptr : nullptr, ws ? ws->bytes : 0, S);
    const int rs = decx_hip_stream_sync(S);
    decx::err::from_hip(&handle, rc != DECX_HIP_OK ? rc : rs, "Linear4");
    return handle;
}

de::DH norm(de::GPU_Matrix& src, de::GPU_Matrix* residual, de::GPU_Vector& weight, de::GPU_Matrix* sum, de::GPU_Matrix& dst, de::GPU_Vector* scales,
            float eps)
{
    de::DH handle; decx::err::success(&handle);
    decx::_GPU_Matrix* x = dynamic_cast<decx::_GPU_Matrix*>(&src);
    decx::_GPU_Matrix* r = dynamic_cast<decx::_GPU_Matrix*>(residual);
    decx::_GPU_Vector* w = dynamic_cast<decx::_GPU_Vector*>(&weight);
    decx::_GPU_Matrix* h = dynamic_cast<decx::_GPU_Matrix*>(sum);
    decx::_GPU_Matrix* y = dynamic_cast<decx::_GPU_Matrix*>(&dst);
    decx::_GPU_Vector* ys = dynamic_cast<decx::_GPU_Vector*>(scales);
    if (!decx::gpu_ready()) return failed(decx::DECX_FAIL_CUDA_not_init, kCudaNotInit);
    if (!x || !w || !y || !x->is_init() || !w->is_init() || (residual && (!r || !r->is_init())) || (sum && !h) || (scales && !ys))
        return failed(decx::DECX_FAIL_CLASS_NOT_INIT, kClassNotInit);
    if ((x->Type() != de::_FP16_ && x->Type() != de::_FP32_) || !whole(x) || !whole(r) || !whole(w)) return failed(decx::DECX_FAIL_UNSUPPORTED_TYPE, kUnsupportedType);
    if (w->Type() != x->Type() || (r && r->Type() != x->Type())) return failed(decx::DECX_FAIL_TYPE_MOT_MATCH, kTypeNotMatch);
    if (w->Len() != x->Width()) return failed(decx::DECX_FAIL_DimsNotMatching, "There must be one weight for every column of the source");
    if (r && (r->Width() != x->Width() || r->Height() != x->Height()))
        return failed(decx::DECX_FAIL_DimsNotMatching, "The source and the residual must be of the same size");
    if (!(eps >= 0.f) || !x->Width() || x->Width() > 0xffff0000u || x->Height() > 0x7fffffffu) return failed(decx::DECX_FAIL_INVALID_PARAM, kInvalidParam);
    // Outputs may lie in the storage of an input of their own shape and type (then the same pitch, and re_construct keeps it),
    // dst in the sum's whatever that was before (both are made that shape), and in nothing else.
    const auto meets = [](const decx::_GPU_Matrix* a, const decx::_GPU_Matrix* b) {
        return a && b && (a == b || (a->is_init() && b->is_init() && a->data() == b->data()));
    };
    const auto same = [&](const decx::_GPU_Matrix* o) { return o->Type() == x->Type() && o->Width() == x->Width() && o->Height() == x->Height(); };
    const bool y_on_input = meets(y, x) || meets(y, r);
    if ((ys && (y_on_input || meets(y, h))) || (y_on_input && !same(y)) || ((meets(h, x) || meets(h, r)) && !same(h)) ||
        (ys && ys->is_init() && ys->data() == w->data()))
        return failed(decx::DECX_FAIL_INVALID_PARAM, kInvalidParam);

    std::lock_guard<std::mutex> guard(decx::module_mutex());
    const uint32_t rows = x->Height(), cols = x->Width();
    if (h && !h->re_construct(x->Type(), cols, rows)) return *de::GetLastError();
    if (!y->re_construct(ys ? de::_UINT8_ : x->Type(), cols, rows)) return *de::GetLastError();
    if (ys && !ys->re_construct(de::_FP32_, rows)) return *de::GetLastError();
    void* S = decx::module_stream();
    int rc;
    if (x->Type() == de::_FP16_)
        rc = decx_hip_rmsnorm_f16((const uint16_t*)x->data(), r ? (const uint16_t*)r->data() : nullptr, (const uint16_t*)w->data(),
                                  h ? (uint16_t*)h->data() : nullptr, y->data(), ys ? (float*)ys->data() : nullptr, rows, cols, x->Pitch(),
                                  r ? r->Pitch() : 0, h ? h->Pitch() : 0, y->Pitch(), eps, S);
    else
        rc = decx_hip_rmsnorm_f32((const float*)x->data(), r ? (const float*)r->data() : nullptr, (const float*)w->data(),
                                  h ? (float*)h->data() : nullptr, y->data(), ys ? (float*)ys->data() : nullptr, rows, cols, x->Pitch(),
                                  r ? r->Pitch() : 0, h ? h->Pitch() : 0, y->Pitch(), eps, S);
    const int rs = decx_hip_stream_sync(S);
    decx::err::from_hip(&handle, rc != DECX_HIP_OK ? rc : rs, "RMSNorm");
    return handle;
}

}  // namespace

_DECX_API_ de::GPU_Matrix4& de::CreateGPUMatrix4Ref() { return *(new decx::_GPU_Matrix4()); }
_DECX_API_ de::GPU_Matrix4* de::CreateGPUMatrix4Ptr() { return new decx::_GPU_Matrix4(); }

_DECX_API_ de::DH de::nn::cuda::Quantize4(de::GPU_Matrix& src, de::GPU_Matrix4& dst, const uint32_t group, const bool zeros)
{
    de::DH handle; decx::err::success(&handle);
    decx::_GPU_Matrix* s = dynamic_cast<decx::_GPU_Matrix*>(&src);
    decx::_GPU_Matrix4* d = dynamic_cast<decx::_GPU_Matrix4*>(&dst);
    if (!decx::gpu_ready()) return failed(decx::DECX_FAIL_CUDA_not_init, kCudaNotInit);
    if (!s || !d || !s->is_init()) return failed(decx::DECX_FAIL_CLASS_NOT_INIT, kClassNotInit);
    if ((s->Type() != de::_FP16_ && s->Type() != de::_FP32_) || !whole(s)) return failed(decx::DECX_FAIL_UNSUPPORTED_TYPE, kUnsupportedType);
    if (!s->Width() || !s->Height() || !decx_hip_q4_scales_count(s->Height(), s->Width(), group)) return failed(decx::DECX_FAIL_INVALID_PARAM, kInvalidParam);
    std::lock_guard<std::mutex> guard(decx::module_mutex());
    if (!d->re_construct(s->Width(), s->Height(), group, zeros)) return failed(decx::DECX_FAIL_CUDA_ALLOCATION, kDevAllocFail);
    void* S = decx::module_stream();
    const int rc = s->Type() == de::_FP16_
        ? decx_hip_q4_quantize_f16((const uint16_t*)s->data(), d->codes(), d->scales(), d->zeros(), s->Height(), s->Width(), s->Pitch(), group, S)
        : decx_hip_q4_quantize_f32((const float*)s->data(), d->codes(), d->scales(), d->zeros(), s->Height(), s->Width(), s->Pitch(), group, S);
    const int rs = decx_hip_stream_sync(S);
    decx::err::from_hip(&handle, rc != DECX_HIP_OK ? rc : rs, "Quantize4");
    return handle;
}

_DECX_API_ de::DH de::nn::cuda::Dequantize4(de::GPU_Matrix4& src, de::GPU_Matrix& dst, const de::_DATA_TYPES_FLAGS_ type)
{
    de::DH handle; decx::err::success(&handle);
    decx::_GPU_Matrix4* s = dynamic_cast<decx::_GPU_Matrix4*>(&src);
    decx::_GPU_Matrix* d = dynamic_cast<decx::_GPU_Matrix*>(&dst);
    if (!decx::gpu_ready()) return failed(decx::DECX_FAIL_CUDA_not_init, kCudaNotInit);
    if (!s || !d || !s->is_init()) return failed(decx::DECX_FAIL_CLASS_NOT_INIT, kClassNotInit);
    if (type != de::_FP16_ && type != de::_FP32_) return failed(decx::DECX_FAIL_UNSUPPORTED_TYPE, kUnsupportedType);
    std::lock_guard<std::mutex> guard(decx::module_mutex());
    if (!d->re_construct(type, s->Width(), s->Height())) return *de::GetLastError();
    void* S = decx::module_stream();
    const int rc = type == de::_FP16_
        ? decx_hip_q4_dequantize_f16(s->codes(), s->scales(), s->zeros(), (uint16_t*)d->data(), s->Height(), s->Width(), d->Pitch(), s->Group(), S)
        : decx_hip_q4_dequantize_f32(s->codes(), s->scales(), s->zeros(), (float*)d->data(), s->Height(), s->Width(), d->Pitch(), s->Group(), S);
    const int rs = decx_hip_stream_sync(S);
    decx::err::from_hip(&handle, rc != DECX_HIP_OK ? rc : rs, "Dequantize4");
    return handle;
}

_DECX_API_ de::DH de::nn::cuda::Linear4(de::GPU_Matrix& src, de::GPU_Matrix4& weights, de::GPU_Matrix& dst, const uint32_t accu)
{
    return linear(src, nullptr, weights, nullptr, dst, nullptr, nullptr, accu);
}
_DECX_API_ de::DH de::nn::cuda::Linear4(de::GPU_Matrix& src, de::GPU_Vector& src_scales, de::GPU_Matrix4& weights, de::GPU_Matrix& dst, const uint32_t accu)
{
    return linear(src, &src_scales, weights, nullptr, dst, nullptr, nullptr, accu);
}
_DECX_API_ de::DH de::nn::cuda::Linear4(de::GPU_Matrix& src, de::GPU_Matrix4& weights, de::GPU_Matrix& C, de::GPU_Matrix& dst, const de::Number alpha,
                                        const de::Number beta)
{
    return linear(src, nullptr, weights, &C, dst, &alpha, &beta, de::Fp16_Accurate_L2);
}
_DECX_API_ de::DH de::nn::cuda::Linear4(de::GPU_Matrix& src, de::GPU_Vector& src_scales, de::GPU_Matrix4& weights, de::GPU_Matrix& C, de::GPU_Matrix& dst,
                                        const de::Number alpha, const de::Number beta)
{
    return linear(src, &src_scales, weights, &C, dst, &alpha, &beta, de::Fp16_Accurate_L2);
}

_DECX_API_ de::DH de::nn::cuda::RMSNorm(de::GPU_Matrix& src, de::GPU_Vector& weight, de::GPU_Matrix& dst, const float eps)
{
    return norm(src, nullptr, weight, nullptr, dst, nullptr, eps);
}
_DECX_API_ de::DH de::nn::cuda::RMSNorm(de::GPU_Matrix& src, de::GPU_Vector& weight, de::GPU_Matrix& dst, de::GPU_Vector& scales, const float eps)
{
    return norm(src, nullptr, weight, nullptr, dst, &scales, eps);
}
_DECX_API_ de::DH de::nn::cuda::RMSNorm(de::GPU_Matrix& src, de::GPU_Matrix& residual, de::GPU_Vector& weight, de::GPU_Matrix& sum, de::GPU_Matrix& dst,
                                        const float eps)
{
    return norm(src, &residual, weight, &sum, dst, nullptr, eps);
}
_DECX_API_ de::DH de::nn::cuda::RMSNorm(de::GPU_Matrix& src, de::GPU_Matrix& residual, de::GPU_Vector& weight, de::GPU_Matrix& sum, de::GPU_Matrix& dst,
                                        de::GPU_Vector& scales, const float eps)
{
    return norm(src, &residual, weight, &sum, dst, &scales, eps);
}
