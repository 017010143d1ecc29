// The forward pass of the root-mean-square norm with an output of 8 bits: the kernels of rms.cuh with a scale per row or per group of 32, 64 or 128 columns.
#include "rms.cuh"

namespace {

template <typename T, int VEC>
void rms_quantised_type(const RmsForward& a, bool wide) {
    if (a.group >= a.n) return wide ? rms_forward_pick<T, VEC, 1>(a) : rms_forward_pick<T, 1, 1>(a);
    if (a.group == 32) wide ? rms_forward_pick<T, VEC, 32>(a) : rms_forward_pick<T, 1, 32>(a);
    else if (a.group == 64) wide ? rms_forward_pick<T, VEC, 64>(a) : rms_forward_pick<T, 1, 64>(a);
    else wide ? rms_forward_pick<T, VEC, 128>(a) : rms_forward_pick<T, 1, 128>(a);
}

}  // namespace

void rms_quantised_run(const RmsForward& a, int type, bool wide) {
    if (type == TB_TYPE_F32) rms_quantised_type<float, 4>(a, wide);
    else if (type == TB_TYPE_F16) rms_quantised_type<__half, 8>(a, wide);
    else rms_quantised_type<__nv_bfloat16, 8>(a, wide);
}
