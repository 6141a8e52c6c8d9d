// The TN form of the FP8 product (see fp8_gemm.cuh).
#include "fp8_gemm.cuh"

namespace ls {

int fp8_launch_tn(bool pair, int bn, bool many, const Fp8Maps &m, const Fp8Params &p, int64_t items, cudaStream_t st)
{
    return launch_form<TN>(pair, bn, many, m, p, items, st);
}

}  // namespace ls
