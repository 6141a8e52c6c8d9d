// The NT form of the FP8 product (see fp8_gemm.cuh).
#include "fp8_gemm.cuh"

namespace ls {

int fp8_launch_nt(bool pair, int bn, bool many, const Fp8Maps &m, const Fp8Params &p, int64_t items, cudaStream_t st)
{
    return launch_form<NT>(pair, bn, many, m, p, items, st);
}

int fp8_cluster_room(int size)
{
    static int room[64][kMaxSplits + 1] = {};
    int dev = 0;
    if (current_device(&dev)) return 0;
    std::lock_guard<std::mutex> lk(state_mutex());
    if (!room[dev][size]) {
        const auto kernel = fp8_gemm_kernel<1, 128, NT, false, true>;
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim.x = unsigned(size), at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(unsigned(size) * 64, 1, 1);
        cfg.blockDim = dim3(kThreads, 1, 1);
        cfg.dynamicSmemBytes = Fp8Cfg<1, 128>::SMEM;
        cfg.attrs = at, cfg.numAttrs = 1;
        int n = 0;
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Fp8Cfg<1, 128>::SMEM) != cudaSuccess ||
            cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) {
            cudaGetLastError();
            return 0;
        }
        room[dev][size] = n;
    }
    return room[dev][size];
}

}  // namespace ls
