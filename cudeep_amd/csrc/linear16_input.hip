// The product dx = dz W of a Linear layer in 16 bits: the kernels of linear16_tile.hpp.
#include "linear16_tile.hpp"

namespace cdx {
namespace l16 {

int run_input(int dtype, const Params& p, const Plan& pl, hipStream_t stream) {
    return with_16(dtype, [&](auto t) { return run<decltype(t), false, true>(p, pl, stream); });
}

}  // namespace l16
}  // namespace cdx
