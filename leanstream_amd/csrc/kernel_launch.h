// A kernel launch that returns its own status: the runtime's last error may be another call's.
#pragma once
#include <hip/hip_runtime.h>
#include <tuple>

namespace lsamd {

template <class... Params, class... Args>
hipError_t launch_kernel(void (*kernel)(Params...), dim3 grid, uint32_t threads, hipStream_t stream, const Args&... args) {
    std::tuple<Params...> values(args...);
    return std::apply(
        [&](Params&... value) {
            void* list[] = {&value...};
            return hipLaunchKernel(reinterpret_cast<const void*>(kernel), grid, dim3(threads), list, 0, stream);
        },
        values);
}

}  // namespace lsamd
