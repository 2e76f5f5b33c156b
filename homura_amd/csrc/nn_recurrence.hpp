// What the recurrence's kernels share: their arguments and one step of the recurrence in either direction.
#pragma once

#include <initializer_list>

#include "nn.hpp"

namespace hmr {
namespace nn {

// A [B, T, C] operand.
struct Sequences {
    char *p;
    int64_t sb, st, sc;
    __device__ __forceinline__ int64_t at(int64_t b, int64_t t, int64_t c) const { return b * sb + t * st + c * sc; }
    template <class T>
    __device__ __forceinline__ T get(int64_t b, int64_t t, int64_t c) const {
        return reinterpret_cast<const T *>(p)[at(b, t, c)];
    }
    template <class T>
    __device__ __forceinline__ void put(int64_t b, int64_t t, int64_t c, T v) const {
        reinterpret_cast<T *>(p)[at(b, t, c)] = v;
    }
};

// A [B, C] operand, or nothing (p null); `wide`: f32 beside 16-bit sequences.
struct States {
    char *p;
    int64_t sb, sc;
    bool wide;
    __device__ __forceinline__ int64_t at(int64_t b, int64_t c) const { return b * sb + c * sc; }
};

struct RecurrenceArgs {
    int64_t B, T, C;
    Sequences gate, input, out;                // forwards
    Sequences grad, state, d_gate, d_input;    // backwards, with gate and input
    bool d_gate_wide;                          // f32 beside 16-bit sequences
    States entry, exit;                        // initial and last; grad_last and d_initial
    States initial;                            // backwards
    const char *lengths;                       // or nullptr
    int64_t lengths_stride;
    bool lengths64;

    // The steps of sequence b, whatever its length says inside 0..T.
    __device__ __forceinline__ int64_t steps(int64_t b) const {
        if (lengths == nullptr) return T;
        const int64_t n = lengths64 ? reinterpret_cast<const int64_t *>(lengths)[b * lengths_stride]
                                    : reinterpret_cast<const int32_t *>(lengths)[b * lengths_stride];
        return n < 0 ? 0 : (n > T ? T : n);
    }
};

// The factor and the addend of a step.
template <class T, int FORM, class C>
__device__ __forceinline__ void factor_and_input(C gate, C input, C &factor, C &addend) {
    if constexpr (FORM == HMN_GATE_FACTOR) {
        factor = gate, addend = input;
    } else {
        C rest;
        sigmoid_pair<T>(gate, factor, rest);
        addend = rest * input;
    }
}

// A step backwards: from the gradient g of the state it led to, the gradients of its gate and input and what is handed
// back to the state before it.
template <class T, int FORM, class C>
__device__ __forceinline__ C step_back(C gate, C input, C g, C before, C &d_gate, C &d_input) {
    if constexpr (FORM == HMN_GATE_FACTOR) {
        d_gate = g * before, d_input = g;
        return gate * g;
    } else {
        C a, rest;
        sigmoid_pair<T>(gate, a, rest);
        const C back = a * g;
        d_input = rest * g;
        d_gate = (before - input) * (back * rest);
        return back;
    }
}

// ---- the scan ------------------------------------------------------------------------------------------------------
//
// Along the direction of processing (q = t forwards, T - 1 - t backwards) every step maps the running value e to
// f e + u: forwards e is the state, f the factor and u the addend; backwards e is the gradient that is handed back,
// f = a_t and u = a_t grad_t. A stretch of steps maps e to F e + U, so stretches fold in any grouping, and each is read
// once: a workgroup holds a tile of R * S steps x L * V channels in registers (lane (r, l) has the S steps from r * S on of
// V channels), folds its steps, then the R slots through LDS, gets the value that enters the tile, and runs its steps
// again from there with the inputs still in registers.
//
// Where there is more than one tile along the sequence, a tile publishes its (F, U) in the workspace, and gets the value
// that enters it by folding, in a fixed order, the tiles before it in its group of about sqrt(tiles) and the groups
// before that. So that every wait ends, tiles are numbered by a ticket that a workgroup draws as it starts, and wait for
// smaller tickets only: their workgroups run already, and publish before they wait. An entry is one 64-bit word (two in
// f64), written and polled with relaxed device-scope atomics, so that no cache has to be flushed; a launch before the
// scan's fills the workspace with words that no entry is.
//
// The memory decides the shape and the order. Tickets follow memory: all of a sequence's channels, then the next steps,
// then the next sequence. A plain kernel that reads two and writes one [8, 2048, 4096] bf16 tensor tile by tile takes
// 86 us when the eight sequences advance together (their rows are 16 MB apart), 72 us in this order, 65 us with rows of
// 512 bytes instead of 256, and 59 us with accesses that pass the caches by.
struct ScanPlan {
    int64_t blocks;  // of channels
    int64_t tiles;   // along the sequence
    int64_t group;   // tiles of a group
    FastDiv by_sequence, by_blocks, by_group;
};

constexpr int kScanBlock = 512;

template <class T, int V, int R, int S>
struct ScanShape {
    static constexpr int kV = V, kR = R, kS = S, kLanes = kScanBlock / R, kChannels = kLanes * V, kSteps = R * S;
    static constexpr int kWords = sizeof(typename Comp<T>::C) / 4;  // 64-bit words of an entry

    static int64_t blocks(int64_t C) { return C / kChannels + (C % kChannels != 0); }
    static int64_t tiles(int64_t steps) { return steps / kSteps + (steps % kSteps != 0); }
    // For no more tiles than a launch has workgroups.
    static ScanPlan plan(int64_t steps, int64_t C) {
        ScanPlan p{};
        p.blocks = blocks(C);
        p.tiles = tiles(steps);
        p.group = 1;
        while (p.group * p.group < p.tiles) ++p.group;
        p.by_sequence = make_fastdiv(static_cast<uint32_t>(p.blocks * p.tiles)), p.by_blocks = make_fastdiv(static_cast<uint32_t>(p.blocks));
        p.by_group = make_fastdiv(static_cast<uint32_t>(p.group));
        return p;
    }
    // 64-bit words of workspace: the ticket's, then the tiles' entries, then the groups'.
    static int64_t words(const ScanPlan &p, int64_t B) {
        return p.tiles <= 1 ? 0 : 8 + B * p.blocks * (p.tiles + p.tiles / p.group + 1) * kChannels * kWords;
    }
};

struct ScanArgs {
    RecurrenceArgs a;
    ScanPlan p;
    uint64_t *room;
};

// The largest tile of any shape in use.
constexpr int64_t kMostSteps = 512, kMostChannels = 256;

// What a scan's launch goes by besides sizes: whether every sequence's channels lie next to each other, and whether every
// row of them begins a cache line.
struct ScanLayout {
    bool adjacent, whole_lines;
};
// Queue the scan of a direction (nn_scan_forward.hip, nn_scan_backward.hip). `room` holds room_for() bytes.
void queue_scan_forward(hipStream_t stream, int32_t dtype, int32_t form, const RecurrenceArgs &a, const ScanLayout &layout, void *room);
void queue_scan_backward(hipStream_t stream, int32_t dtype, int32_t form, const RecurrenceArgs &a, const ScanLayout &layout, void *room);
// Sequences of so few steps go a thread per channel: there is nothing to gain in a scan of up to eight ([64, 6, 4096] bf16
// 5 us, 10 by a scan), nor of up to 32 where there are enough channels to keep the chip busy, 2^16 of all sequences
// ([512, 24, 4096] bf16 95 us and 167, backwards 145 and 315; [4096, 16, 40] 7 and 18; but [512, 64, 4096] bf16 248 and 186).
constexpr int64_t kFewSteps = 8, kFewWithMany = 32, kMany = int64_t{1} << 16;
// Of those, 13 to 16 steps make a nearly full tile of the shortest shape, and where rows fill its lanes (a tenth idle at most)
// and every operand is 64 MB or more, wide accesses are worth the fold: f32 [512, 16, 4096] 73 us and a thread per channel 87,
// backwards 142 and 161; backwards in 16 bits too, [512, 16, 4096] bf16 82 and 101, [2000, 13, 1003] 81 and 84. Not forwards
// (52 and 42), smaller ([128, 16, 4096] f32 backwards 34 and 32) or with idle lanes ([8000, 16, 260] bf16 backwards 139 and
// 117).
constexpr int64_t kNearlyATile = 13, kLarge = int64_t{64} << 20;
bool short_scan_used(const hmr_tensor_desc *gate, const ScanLayout &layout, bool backward);
// Whether the sequences are long enough for a scan, and not too many for a launch with a workgroup for every tile.
bool scan_used(const hmr_tensor_desc *gate);
// Bytes of workspace of either direction, whatever the operands' strides.
int64_t room_for(const hmr_tensor_desc *gate);

}  // namespace nn
}  // namespace hmr
