// fp16_pair.hpp - a float as the sum of two fp16 values.
#pragma once

#include "sdh_internal.hpp"

namespace sdh {
namespace {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));

// Two floats of magnitude below 2^16 into hi + lo: hi is p towards zero in fp16
// (v_cvt_pkrtz), lo = p - hi rounded to fp16 (|lo| < 2^-10 p, so the pair is
// within 2^-21 p; below 2^-14, where fp16 is subnormal, within 2^-25
// absolutely). v_fma_mixlo/mixhi take hi's half as it lies in the packed pair and
// round the exact difference into a half: three instructions a pair, where
// masking, subtracting and packing took six.
__device__ __forceinline__ void split_pair(float p0, float p1, h2& hi, h2& lo) {
    hi = __builtin_bit_cast(h2, __builtin_amdgcn_cvt_pkrtz(p0, p1));
    const unsigned h = __builtin_bit_cast(unsigned, hi);
    unsigned l;
    asm("v_fma_mixlo_f16 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(l) : "v"(h), "v"(p0));
    asm("v_fma_mixhi_f16 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "+v"(l) : "v"(h), "v"(p1));
    lo = __builtin_bit_cast(h2, l);
}

}  // namespace
}  // namespace sdh
