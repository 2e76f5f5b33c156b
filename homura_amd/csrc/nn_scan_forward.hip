// The scan's kernels, forwards.
#include "nn_scan.hpp"

namespace hmr {
namespace nn {

void queue_scan_forward(hipStream_t stream, int32_t dtype, int32_t form, const RecurrenceArgs &a, const ScanLayout &layout, void *room) {
    queue_scan<false>(stream, dtype, form, a, layout, room);
}

namespace {

// The most that any shape makes of measure(shape).
template <class F>
int64_t most_of(const hmr_tensor_desc *gate, F measure) {
    int64_t most = 0;
    with_float_type(gate->dtype, [&](auto tag) {
        with_scan_shapes<typename decltype(tag)::type>(gate->sizes[1], [&](auto shape) {
            const int64_t x = measure(shape);
            if (x > most) most = x;
        });
    });
    return most;
}

}  // namespace

bool scan_used(const hmr_tensor_desc *gate) {
    if (gate->sizes[0] == 0 || gate->sizes[2] == 0 || gate->sizes[1] <= kFewSteps) return false;
    if (gate->sizes[1] <= kFewWithMany && gate->sizes[0] >= (kMany + gate->sizes[2] - 1) / gate->sizes[2]) return false;
    return fits_launch(most_of(gate,
                               [&](auto shape) {
                                   using Shape = decltype(shape);
                                   return gate->sizes[0] * Shape::blocks(gate->sizes[2]) * Shape::tiles(gate->sizes[1]);
                               }),
                       kScanBlock);
}

bool short_scan_used(const hmr_tensor_desc *gate, const ScanLayout &layout, bool backward) {
    const int64_t B = gate->sizes[0], T = gate->sizes[1], C = gate->sizes[2], size = dtype_size(gate->dtype);
    if (!layout.adjacent || T < kNearlyATile || T > kShortest || size > 4 || (size == 2 && !backward)) return false;
    bool used = false;
    with_float_type(gate->dtype, [&](auto tag) {
        using Shape = ShortShape<typename decltype(tag)::type>;
        const int64_t blocks = Shape::blocks(C);
        used = B * T * C * size >= kLarge && 10 * C >= 9 * blocks * Shape::kChannels && fits_launch(B * blocks, kScanBlock);
    });
    return used;
}

int64_t room_for(const hmr_tensor_desc *gate) {
    if (!scan_used(gate)) return 0;
    return 8 * most_of(gate, [&](auto shape) {
        using Shape = decltype(shape);
        return Shape::words(Shape::plan(gate->sizes[1], gate->sizes[2]), gate->sizes[0]);
    });
}

}  // namespace nn
}  // namespace hmr
