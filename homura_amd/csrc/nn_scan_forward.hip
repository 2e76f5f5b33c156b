// The scan's kernels, forwards.
#include "nn_scan.hpp"

namespace hmr {
namespace nn {

void queue_scan_forward(hipStream_t stream, int32_t dtype, int32_t form, const RecurrenceArgs &a, bool vectors, void *room) {
    queue_scan<false>(stream, dtype, form, a, vectors, room);
}

int64_t room_for(const hmr_tensor_desc *gate) {
    const int64_t B = gate->sizes[0], T = gate->sizes[1], C = gate->sizes[2];
    if (B * C == 0) return 0;
    switch (gate->dtype) {
        case HMR_F16: return scan_room<f16_t>(B, T, C);
        case HMR_BF16: return scan_room<bf16_t>(B, T, C);
        case HMR_F32: return scan_room<float>(B, T, C);
        default: return scan_room<double>(B, T, C);
    }
}

}  // namespace nn
}  // namespace hmr
