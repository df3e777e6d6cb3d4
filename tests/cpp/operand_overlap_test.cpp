// The rules of decx_amd/csrc/operand_overlap.hpp: every pair that must not be one buffer, and the pairs that may.
#include "../../decx_amd/csrc/operand_overlap.hpp"

#include <cstdio>

using namespace decx_hip;

static int failures = 0;
#define CHECK(cond) do { if (!(cond)) { ++failures; std::printf("FAILED line %d: %s\n", __LINE__, #cond); } } while (0)

int main()
{
    char at[8] = {};
    enum { X, XS, CODES, SCALES, ZEROS, C, Y, WS, COUNT };
    const auto product = [&](int a, int b) {               // with operand b in the place of a
        const void* p[COUNT];
        for (int i = 0; i < COUNT; ++i) p[i] = at + i;
        if (a >= 0) p[b] = p[a];
        return product_operands_apart(p[X], p[XS], p[CODES], p[SCALES], p[ZEROS], p[C], p[Y], p[WS]);
    };
    CHECK(product(-1, -1));
    for (int in : {X, XS, CODES, SCALES, ZEROS}) { CHECK(!product(in, Y)); CHECK(!product(in, WS)); }
    CHECK(!product(C, WS) && !product(Y, WS));
    CHECK(product(C, Y));                                  // the residual in place
    CHECK(product(X, C) && product(SCALES, ZEROS));        // inputs among themselves
    CHECK(product_operands_apart(at, nullptr, at + 1, at + 2, nullptr, nullptr, at + 3, nullptr));
    CHECK(product_operands_apart(nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, at, nullptr));      // K = 0
    CHECK(!product_operands_apart(at, nullptr, at + 1, at + 2, nullptr, nullptr, at, nullptr));

    for (int a = 0; a < 4; ++a)
        for (int b = 0; b < a; ++b) {
            const void* p[4] = {at, at + 1, at + 2, at + 3};
            CHECK(quantize_operands_apart(p[0], p[1], p[2], p[3]) && dequantize_operands_apart(p[0], p[1], p[2], p[3]));
            p[a] = p[b];
            CHECK(!quantize_operands_apart(p[0], p[1], p[2], p[3]));
            CHECK(dequantize_operands_apart(p[0], p[1], p[2], p[3]) == (b != 0));
        }
    CHECK(quantize_operands_apart(at, at + 1, at + 2, nullptr) && dequantize_operands_apart(at, at + 1, at + 2, nullptr));
    if (!failures) std::puts("all ok");
    return failures != 0;
}
