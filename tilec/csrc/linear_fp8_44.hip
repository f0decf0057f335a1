// x in e4m3, w in e4m3.
#include "linear_fp8_kernels.h"

namespace tilec {
template hipError_t launch_fp8<0, 0>(const Fp8Args&, bool, int, int, hipStream_t);
}
