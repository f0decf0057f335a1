// x in e5m2, w in e5m2.
#include "linear_fp8_kernels.h"

namespace tilec {
template hipError_t launch_fp8<1, 1>(const Fp8Args&, bool, int, int, hipStream_t);
}
