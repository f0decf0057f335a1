// x in e4m3, w in e5m2.
#include "linear_fp8_kernels.h"

namespace tilec {
template hipError_t launch_fp8<0, 1>(const Fp8Args&, bool, int, int, hipStream_t);
}
