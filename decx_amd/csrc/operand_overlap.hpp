// Host-side checks that no output of a call with 4-bit weights lies where an input does.  Pointers are compared, not ranges:
// a result may share rows with its source (columns side by side of one wide matrix), so ranges that meet prove nothing, and
// the same first element always does.  (No HIP in here: the rules are tested on the CPU.)
#pragma once
#include <cstdint>
#include <initializer_list>

namespace decx_hip {

inline bool one_of(const void* p, std::initializer_list<const void*> others)
{
    if (!p) return false;
    for (const void* o : others) if (o == p) return true;
    return false;
}

// A product: workgroups read X, its factors and the weights while others store Y already, and the workspace is written before
// Y is.  (C may be Y, at its pitch: every element is read by the thread that writes it.)  `workspace` is null where none is
// used, X and the weights where K = 0.
inline bool product_operands_apart(const void* X, const void* x_scales, const void* codes, const void* scales, const void* zeros, const void* C,
                                   const void* Y, const void* workspace)
{
    return !one_of(Y, {X, x_scales, codes, scales, zeros}) && !one_of(workspace, {X, x_scales, codes, scales, zeros, C, Y});
}

// W to 4 bits (the parts are outputs) and back (W is): no output in the place of anything else.
inline bool quantize_operands_apart(const void* W, const void* codes, const void* scales, const void* zeros)
{
    return !one_of(W, {codes, scales, zeros}) && !one_of(codes, {scales, zeros}) && !one_of(scales, {zeros});
}
inline bool dequantize_operands_apart(const void* W, const void* codes, const void* scales, const void* zeros) { return !one_of(W, {codes, scales, zeros}); }

}  // namespace decx_hip
