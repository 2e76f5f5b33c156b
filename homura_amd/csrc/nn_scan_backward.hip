// The scan's kernels, backwards.
#include "nn_scan.hpp"

namespace hmr {
namespace nn {

void queue_scan_backward(hipStream_t stream, int32_t dtype, int32_t form, const RecurrenceArgs &a, const ScanLayout &layout, void *room) {
    queue_scan<true>(stream, dtype, form, a, layout, room);
}

}  // namespace nn
}  // namespace hmr
