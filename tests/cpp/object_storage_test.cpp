// Storage of the classes behind the de:: objects when they are made anew (no GPU; linked with their sources).
#include "decx_internal.hpp"

#include <iostream>

static int g_failures = 0;
#define CHECK(cond) do { if (!(cond)) { ++g_failures; std::cerr << "FAILED line " << __LINE__ << ": " #cond "\n"; } } while (0)

int main()
{
    // a matrix that was given a type of larger elements has no room for them at its size
    decx::_Matrix m(de::_FP16_, 64, 4, de::_NA_);
    m.Reinterpret(de::_FP32_);
    m.re_construct(de::_FP32_, 64, 4);
    CHECK(m.Type() == de::_FP32_ && m.get_layout()._single_element_size == 4 && m.total_bytes() >= 64 * 4 * 4);
    for (int r = 0; r < 4; ++r) for (int c = 0; c < 64; ++c) *m.ptr<float>(r, c) = 1.f;
    decx::_Vector v(de::_FP16_, 100);
    v.Reinterpret(de::_FP32_);
    CHECK(v.re_construct(de::_FP32_, 100) && v.element_bytes() == 4 && v.capacity_bytes() >= 400);
    // an alias of it knows what is there
    decx::_Matrix r(de::_FP16_, 64, 4, de::_NA_), alias;
    r.Reinterpret(de::_FP32_);
    alias.SoftCopy(r);
    CHECK(alias.Type() == de::_FP32_ && alias.total_bytes() == r.total_bytes() && alias.Pitch() == r.Pitch() && alias.get_layout()._single_element_size == 2);
    decx::_Vector rv(de::_FP16_, 100), valias;
    rv.Reinterpret(de::_FP32_);
    valias.SoftCopy(rv);
    CHECK(valias.Type() == de::_FP32_ && valias.element_bytes() == 2 && valias.Len() == 100 && valias.data() == rv.data());
    // the same type and size again keeps it
    void* const at = m.data();
    m.re_construct(de::_FP32_, 64, 4);
    CHECK(m.data() == at);

    // no memory to be had (no device): what the object was it stays
    decx::_GPU_Matrix g;
    CHECK(!g.re_construct(de::_FP32_, 64, 4) && g.Type() == de::_VOID_ && g.Width() == 0 && g.Height() == 0 && !g.is_init());
    decx::_GPU_Vector gv;
    CHECK(!gv.re_construct(de::_FP32_, 100) && gv.Type() == de::_VOID_ && gv.Len() == 0 && !gv.is_init());
    return g_failures != 0;
}
