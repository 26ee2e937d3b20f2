// Instances of the block-scaled product of few rows.
#include "f8_gemm_few.h"

namespace acc950 {
namespace {

template <int TM, int TN, int CW, int KW, int DEPTH>
hipError_t run(const F8GemmArgs& a, bool wide, hipStream_t s)
{
    if (a.offsets) return wide ? launch_f8_few<F8FewConfig<TM, TN, CW, KW, DEPTH, true, false, true, false>>(a, s)
                               : launch_f8_few<F8FewConfig<TM, TN, CW, KW, DEPTH, false, false, true, false>>(a, s);
    if (a.group_shift == 0) return wide ? launch_f8_few<F8FewConfig<TM, TN, CW, KW, DEPTH, true, true, false, false>>(a, s)
                                        : launch_f8_few<F8FewConfig<TM, TN, CW, KW, DEPTH, false, true, false, false>>(a, s);
    return wide ? launch_f8_few<F8FewConfig<TM, TN, CW, KW, DEPTH, true, false, false, false>>(a, s)
                : launch_f8_few<F8FewConfig<TM, TN, CW, KW, DEPTH, false, false, false, false>>(a, s);
}

} // namespace

hipError_t launch_f8_gemm_few(const F8GemmArgs& a, int form, bool wide, hipStream_t s)
{
    return form == 0 ? run<1, 1, 1, 4, 4>(a, wide, s) : run<1, 2, 4, 1, 4>(a, wide, s);
}

hipError_t launch_f8_gated_few(const F8GemmArgs& a, hipStream_t s) { return launch_f8_few<F8FewConfig<1, 2, 8, 1, 4, true, false, true, true>>(a, s); }

} // namespace acc950
