// Translation unit of the kernels for few query rows on a shared prefix and own keys, for one 16-bit element type
// (-DNA2D_TC_DT=1: bf16, 2: fp16).
#include "na2d_prefix_tokens.cuh"

namespace na2d_prefix {

#if NA2D_TC_DT == 1
#define NA2D_TC_TYPE __nv_bfloat16
#define NA2D_TC_NAME(base) base##_bf16
#elif NA2D_TC_DT == 2
#define NA2D_TC_TYPE __half
#define NA2D_TC_NAME(base) base##_f16
#else
#error "compile with -DNA2D_TC_DT=1 (bf16) or 2 (fp16)"
#endif

namespace {

template <int D, int MT>
int launch_line(const Place& at, const Tokens& x) {
    auto kern = prefix_tokens_kernel<NA2D_TC_TYPE, D, MT>;
    static std::atomic<unsigned long long> opted{0};
    if (na2d_tc::opt_in_smem(kern, kTokenSmem<D>, at.device, opted) != cudaSuccess) return NA2D_ERR_CUDA;
    *at.launched += 1;
    return na2d_launch::launch(true, kern, (unsigned)na2d_tc::sm_count(at.device), kTokenThreads, kTokenSmem<D>, at.st, x) == cudaSuccess
               ? NA2D_OK
               : NA2D_ERR_CUDA;
}
template <int D>
int by_rows(const Place& at, const Tokens& x) {
    const int rows = std::max(x.side[0].entries ? x.side[0].rows : 0, x.side[1].entries ? x.side[1].rows : 0);
    if (rows <= 16) return launch_line<D, 1>(at, x);
    if (rows <= 32) return launch_line<D, 2>(at, x);
    return NA2D_ERR_UNSUPPORTED;
}
}  // namespace

int NA2D_TC_NAME(tokens)(const Place& at, const Tokens& x, const JoinPrefix& prefix, void* o, float* lse, int B) {
    const int rc = x.C <= 32 ? by_rows<32>(at, x) : x.C <= 64 ? by_rows<64>(at, x) : by_rows<128>(at, x);
    if (rc != NA2D_OK) return rc;
    const long long rows = (long long)B * x.N * x.Tq;
    if (rows > 0x7fffffffLL) return NA2D_ERR_TOO_LARGE;
    *at.launched += 1;
    return na2d_launch::launch(true, prefix_join_kernel<NA2D_TC_TYPE>, (unsigned)rows, 128, 0, at.st, x, prefix, (NA2D_TC_TYPE*)o, lse) == cudaSuccess
               ? NA2D_OK
               : NA2D_ERR_CUDA;
}

}  // namespace na2d_prefix
