// gemv_mfma_kernel, all six formats.
#include "gemv_mfma.h"
#include "tu.h"

namespace jitnn {

template <int FMT>
static KernelRef ref(bool epilogue) {
    return {epilogue ? (const void *)gemv_mfma_epilogue_kernel<FMT> : (const void *)gemv_mfma_kernel<FMT>, gemv_mfma_lds_bytes<FMT>()};
}

KernelRef gemv_mfma_kernel_ref(int fmt, bool epilogue) {
    switch (fmt) {
    case F_Q4_0: return ref<F_Q4_0>(epilogue);
    case F_Q4_1: return ref<F_Q4_1>(epilogue);
    case F_Q8_0: return ref<F_Q8_0>(epilogue);
    case F_Q4_K: return ref<F_Q4_K>(epilogue);
    case F_Q5_K: return ref<F_Q5_K>(epilogue);
    case F_Q6_K: return ref<F_Q6_K>(epilogue);
    default: return {nullptr, 0};
    }
}

template <int FMT>
static void launch(unsigned blocks, hipStream_t s, const uint8_t *W, const float *x, const float *bias, const Epilogue &e, float *y, int n, int k, int rows) {
    if (e.any()) hipLaunchKernelGGL(gemv_mfma_epilogue_kernel<FMT>, dim3(blocks), dim3(MF_THREADS), gemv_mfma_lds_bytes<FMT>(), s, W, x, bias, y, n, k, rows, (int)blocks, e);
    else hipLaunchKernelGGL(gemv_mfma_kernel<FMT>, dim3(blocks), dim3(MF_THREADS), gemv_mfma_lds_bytes<FMT>(), s, W, x, bias, y, n, k, rows, (int)blocks);
}

void gemv_mfma_launch(int fmt, unsigned blocks, hipStream_t s, const uint8_t *W, const float *x, const float *bias, const Epilogue &e, float *y, int n, int k, int rows) {
    switch (fmt) {
    case F_Q4_0: launch<F_Q4_0>(blocks, s, W, x, bias, e, y, n, k, rows); break;
    case F_Q4_1: launch<F_Q4_1>(blocks, s, W, x, bias, e, y, n, k, rows); break;
    case F_Q8_0: launch<F_Q8_0>(blocks, s, W, x, bias, e, y, n, k, rows); break;
    case F_Q4_K: launch<F_Q4_K>(blocks, s, W, x, bias, e, y, n, k, rows); break;
    case F_Q5_K: launch<F_Q5_K>(blocks, s, W, x, bias, e, y, n, k, rows); break;
    case F_Q6_K: launch<F_Q6_K>(blocks, s, W, x, bias, e, y, n, k, rows); break;
    default: break;
    }
}

}  // namespace jitnn
