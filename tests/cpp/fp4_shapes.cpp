// The C++ host mirror's 4-bit operands of sizes that do not fit (staleynet_cuda.hpp): refused where they are
// made, not allocated by what is left of the size.
#include <cstdio>

#include "staleynet_cuda.hpp"

using namespace staleynet_cuda;

template <class Make>
static bool refused(Make&& make) {
    try {
        make();
    } catch (const Panic& panic) {
        return panic.status == SN_ERR_OVERFLOW;
    }
    return false;
}

int main() {
    const Gpu gpu = Gpu::new_(0);
    const size_t half = size_t(1) << 32;
    bool ok = refused([&] { gpu.fp4_cache(sn_fp4_cache_shape{half, half, 1, 64}); });
    ok &= refused([&] { gpu.fp4_cache(sn_fp4_cache_shape{1, half, half + 1, 64}); });
    ok &= refused([&] { gpu.fp4_matrix(half, half * 32); });
    const Fp4Cache cache = gpu.fp4_cache(sn_fp4_cache_shape{2, 3, 5, 64});
    ok &= cache.k_codes.len() == 2 * 3 * 5 * 32 && cache.v_scales.len() == 2 * 3 * 5 * 2;
    std::printf(ok ? "fp4 shapes ok\n" : "a size was not refused, or a cache has another\n");
    return ok ? 0 : 1;
}
