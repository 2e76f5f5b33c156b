// The scan's kernels (nn_recurrence.hpp says how a tile gets the value that enters it, and why its shape).
#pragma once

#include "nn_recurrence.hpp"

namespace hmr {
namespace nn {

constexpr uint64_t kNoEntry = ~uint64_t{0};

// Lays the workspace of a chained scan out: no entries, the ticket at zero.
static __global__ void __launch_bounds__(kBlock) scan_clear_kernel(uint64_t *room, int64_t words) {
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x; i < words; i += static_cast<int64_t>(gridDim.x) * kBlock) {
        room[i] = i < 8 ? 0 : kNoEntry;
    }
}

// An entry, the map e -> f e + u, in words of which none is kNoEntry (only a NaN could be).
__device__ __forceinline__ void publish(uint64_t *p, float f, float u) {
    uint64_t w = (static_cast<uint64_t>(bits_as<uint32_t>(u)) << 32) | bits_as<uint32_t>(f);
    if (w == kNoEntry) w = 0x7FC000007FC00000ull;
    __hip_atomic_store(p, w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void publish(uint64_t *p, double f, double u) {
    const double v[2] = {f, u};
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        uint64_t w = bits_as<uint64_t>(v[k]);
        if (w == kNoEntry) w = 0x7FF8000000000000ull;
        __hip_atomic_store(p + k, w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
}
__device__ __forceinline__ uint64_t peek(const uint64_t *p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ uint64_t await(const uint64_t *p, uint64_t w) {
    while (w == kNoEntry) {
        __builtin_amdgcn_s_sleep(1);
        w = peek(p);
    }
    return w;
}

// f e + u; a stretch whose factors' product overflowed still leaves a zero what it is.
template <class C>
__device__ __forceinline__ C carried(C f, C e, C u) {
    return e == C(0) ? u : fma_(f, e, u);
}

// Folds `count` published entries of this thread's channel, in order, onto (f, u): the first one's word is p[at], each
// next one `apart` words on.
template <class C>
__device__ __forceinline__ void fold_entries(const uint64_t *p, uint32_t at, uint32_t apart, uint32_t count, C &f, C &u) {
    constexpr uint32_t kAhead = 4, W = sizeof(C) / 4;
    for (uint32_t i = 0; i < count; i += kAhead) {
        uint64_t w[kAhead][W];
#pragma unroll
        for (uint32_t j = 0; j < kAhead; ++j) {
            if (i + j < count) {
                const uint64_t *q = p + static_cast<uint64_t>(i + j) * apart;
#pragma unroll
                for (uint32_t k = 0; k < W; ++k) w[j][k] = peek(q + (at + k));
            }
        }
#pragma unroll
        for (uint32_t j = 0; j < kAhead; ++j) {
            if (i + j < count) {
                const uint64_t *q = p + static_cast<uint64_t>(i + j) * apart;
                C ef, eu;
                if constexpr (W == 1) {
                    const uint64_t x = await(q + at, w[j][0]);
                    ef = bits_as<float>(static_cast<uint32_t>(x)), eu = bits_as<float>(static_cast<uint32_t>(x >> 32));
                } else {
                    ef = bits_as<double>(await(q + at, w[j][0])), eu = bits_as<double>(await(q + (at + 1), w[j][1]));
                }
                u = carried(ef, u, eu);
                f *= ef;
            }
        }
    }
}

template <class T, class Shape, int FORM, bool BACK, bool CHAIN, int PASSING>
__global__ void __launch_bounds__(kScanBlock) scan_kernel(ScanArgs s) {
    using C = typename Comp<T>::C;
    constexpr int V = Shape::kV, R = Shape::kR, S = Shape::kS;
    constexpr int L = Shape::kLanes, CL = Shape::kChannels, TT = Shape::kSteps, W = Shape::kWords;
    static_assert(TT <= kMostSteps && CL <= kMostChannels, "spans the host checks for");
    static_assert(2 * CL <= kScanBlock, "a thread per channel folds slots and tiles, another one groups");
    constexpr bool kLoadPast = PASSING == kPastCaches, kStorePast = PASSING != kThroughCaches;
    // Many slots fold in two steps, runs of them by a thread each first.
    constexpr int P = R > 32 ? 16 : R, RP = R / P;
    static_assert(RP == 1 || P * CL <= kScanBlock, "a thread per channel and run of slots");
    __shared__ C slot_f[R][CL], slot_u[R][CL];
    __shared__ C run_f[RP > 1 ? P : 1][CL], run_u[RP > 1 ? P : 1][CL];
    __shared__ C before_group[CHAIN ? CL : 1];
    __shared__ uint32_t drawn;
    const RecurrenceArgs &a = s.a;
    const int tid = threadIdx.x, l = tid % L, r = tid / L;

    struct Raw {
        Vec<T, V> gate[S], input[S], grad[BACK ? S : 1], before[BACK ? S : 1];
    };
    auto clamped = [](int64_t n) { return static_cast<int>(n < 0 ? 0 : (n > S ? S : n)); };
    // Where a tile lies.
    struct Tile {
        int64_t b, k, block;
        int64_t steps;   // of its sequence
        int64_t c0, c1;  // the block's channels
        bool lane_on;    // whether the lane has channels,
        int at;          // and its first one's place in the block
        // The lane's steps from `from` to `to` lie inside the sequence, those from `end` on past the batch's last; `first`
        // is the sequence's first step (if it is the lane's at all), which backwards starts from `initial`.
        int from, to, end, first;
        __device__ __forceinline__ bool has(int i) const { return i >= from && i < to; }
    };
    auto find = [&](uint32_t ticket) {
        Tile t;
        t.b = divide(ticket, s.p.by_sequence);
        const int64_t of_sequence = ticket - t.b * (s.p.blocks * s.p.tiles);
        t.k = divide(static_cast<uint32_t>(of_sequence), s.p.by_blocks), t.block = of_sequence - t.k * s.p.blocks;
        t.steps = a.steps(t.b);
        // A vector never crosses the last channel: the last block begins early enough to have one, and the block before it
        // ends there, so that no channel is two workgroups' (a state may be read and written in one place). Inside a
        // block the last lane's vector moves back over its neighbour's channels, and both compute the same for those.
        const int64_t last = V > 1 && (s.p.blocks - 1) * CL > a.C - V ? a.C - V : (s.p.blocks - 1) * CL;  // block's first channel
        t.c0 = t.block + 1 < s.p.blocks ? t.block * CL : last;
        t.c1 = t.block + 1 < s.p.blocks ? (t.c0 + CL < last ? t.c0 + CL : last) : a.C;
        t.lane_on = t.c0 + l * V < t.c1;
        const int64_t c = V > 1 && t.c0 + l * V > t.c1 - V ? t.c1 - V : t.c0 + l * V;
        t.at = static_cast<int>(c - t.c0);
        const int64_t q0 = t.k * TT + r * S;
        t.end = clamped(a.T - q0);
        t.from = BACK ? clamped(a.T - t.steps - q0) : 0, t.to = BACK ? t.end : clamped(t.steps - q0);
        t.first = BACK && a.T - q0 <= S ? static_cast<int>(a.T - 1 - q0) : S;
        return t;
    };
    // The address of a tile's earliest step (less `back`) and first channel, the same for the whole workgroup, and the
    // lane's offset from there to its own earliest step in 32 bits (the host has checked that a tile spans less); step i
    // of the lane is a number of steps on that is the same for the whole workgroup again.
    auto base_of = [&](const Tile &t, const Sequences &x, int back, int64_t size) {
        const int64_t first = BACK ? a.T - (t.k + 1) * TT : t.k * TT;
        return x.p + (t.b * x.sb + (first - back) * x.st + t.c0 * x.sc) * size;
    };
    auto row_of = [&](char *from, const Tile &t, const Sequences &x, int i, uint32_t size) {
        const int lane_step = BACK ? TT - S - r * S : r * S, step = BACK ? S - 1 - i : i;
        const uint32_t off = (static_cast<uint32_t>(lane_step) * static_cast<uint32_t>(x.st) + static_cast<uint32_t>(t.at) * static_cast<uint32_t>(x.sc)) * size;
        return from + step * x.st * static_cast<int64_t>(size) + off;
    };
    auto base = [&](const Tile &t, const Sequences &x, int back = 0) { return base_of(t, x, back, sizeof(T)); };
    auto row = [&](char *from, const Tile &t, const Sequences &x, int i) { return reinterpret_cast<T *>(row_of(from, t, x, i, sizeof(T))); };
    // Steps outside the sequence get what maps a value to itself: a factor of one (sigmoid's at infinity) and nothing to add.
    auto load = [&](const Tile &t, Raw &raw) {
        char *gate = base(t, a.gate), *input = nullptr, *grad = nullptr, *before = nullptr;
        if constexpr (!BACK || FORM == HMN_GATE_SIGMOID) input = base(t, a.input);
        if constexpr (BACK) grad = base(t, a.grad), before = base(t, a.state, 1);
#pragma unroll
        for (int i = 0; i < S; ++i) {
            raw.gate[i].fill(FORM == HMN_GATE_FACTOR ? C(1) : C(__builtin_inf()));
            raw.input[i].fill(C(0));
            if constexpr (BACK) raw.grad[i].fill(C(0)), raw.before[i].fill(C(0));
            if (t.lane_on && t.has(i)) {
                raw.gate[i].template load<kLoadPast>(row(gate, t, a.gate, i));
                if constexpr (!BACK || FORM == HMN_GATE_SIGMOID) raw.input[i].template load<kLoadPast>(row(input, t, a.input, i));
                if constexpr (BACK) {
                    raw.grad[i].template load<kLoadPast>(row(grad, t, a.grad, i));
                    if (i != t.first) raw.before[i].template load<kLoadPast>(row(before, t, a.state, i));
                }
            }
        }
    };
    uint32_t ticket = blockIdx.x;
    if constexpr (CHAIN) {
        if (tid == 0) drawn = atomicAdd(reinterpret_cast<uint32_t *>(s.room), 1u);
        __syncthreads();
        ticket = __builtin_amdgcn_readfirstlane(drawn);
    }
    const Tile t = find(ticket);
    Raw now;
    load(t, now);
    const int64_t cj = t.c0 + tid;  // the channel whose slots this thread folds
    const bool folds = tid < CL && cj < t.c1;
    C carry = 0;  // of channel cj: the value that enters the tile, then the one that leaves it
    if (folds && t.k == 0 && a.entry.p != nullptr) carry = load_state<T>(a.entry.p, a.entry.at(t.b, cj), a.entry.wide);
    // The lane's steps as maps, and their fold: what it adds is the state from zero exactly as steps one by one leave it (a
    // zero times a factor that is not finite is NaN, so that what follows such a step is never finite, though steps from
    // another state might leave an infinity where the fold has NaN). The maps are computed again when the steps are run.
    auto map = [&](int i, int j, C &f, C &add) {
        const C z = now.gate[i].get(j);
        if constexpr (!BACK) {
            factor_and_input<T, FORM>(z, now.input[i].get(j), f, add);
        } else {
            C rest;
            if constexpr (FORM == HMN_GATE_SIGMOID) sigmoid_pair<T>(z, f, rest);
            else f = z;
            add = f * now.grad[i].get(j);
        }
    };
    C fold_f[V], fold_u[V];
#pragma unroll
    for (int i = 0; i < S; ++i) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            C f, add;
            map(i, j, f, add);
            fold_u[j] = fma_(f, i == 0 ? C(0) : fold_u[j], add);
            fold_f[j] = i == 0 ? f : fold_f[j] * f;
        }
    }
#pragma unroll
    for (int i = 0; i < S; ++i) {
        now.gate[i].forget();
        if constexpr (!BACK) now.input[i].forget();
        else now.grad[i].forget();
    }
    if (t.lane_on) {
#pragma unroll
        for (int j = 0; j < V; ++j) slot_f[r][t.at + j] = fold_f[j], slot_u[r][t.at + j] = fold_u[j];
    }
    __syncthreads();
    // The maps of this thread's channel: of the runs of slots, or of the slots themselves.
    auto part_f = [&](int i) -> C & {
        if constexpr (RP > 1) return run_f[i][tid];
        else return slot_f[i][tid];
    };
    auto part_u = [&](int i) -> C & {
        if constexpr (RP > 1) return run_u[i][tid];
        else return slot_u[i][tid];
    };
    const int run_channel = tid % CL, run = tid / CL;
    const bool has_run = RP > 1 && run < P && t.c0 + run_channel < t.c1;
    if constexpr (RP > 1) {
        if (has_run) {
            C f = slot_f[run * RP][run_channel], u = slot_u[run * RP][run_channel];
#pragma unroll
            for (int i = 1; i < RP; ++i) {
                const C nf = slot_f[run * RP + i][run_channel];
                u = carried(nf, u, slot_u[run * RP + i][run_channel]);
                f *= nf;
            }
            run_f[run][run_channel] = f, run_u[run][run_channel] = u;
        }
        __syncthreads();
    }
    if constexpr (CHAIN) {
        const int64_t g = divide(static_cast<uint32_t>(t.k), s.p.by_group), first = g * s.p.group, chain = t.b * s.p.blocks + t.block;
        uint64_t *entries = s.room + 8 + chain * s.p.tiles * CL * W;
        uint64_t *groups = s.room + 8 + (a.B * s.p.blocks * s.p.tiles + chain * (s.p.tiles / s.p.group + 1)) * CL * W;
        C group_f = 1, group_u = 0;
        if (folds) {
            C tile_f = part_f(0), tile_u = part_u(0);
#pragma unroll 8
            for (int i = 1; i < P; ++i) {
                const C nf = part_f(i);
                tile_u = carried(nf, tile_u, part_u(i));
                tile_f *= nf;
            }
            // The first tile knows what enters it: its map is constant, and no other tile reads `entry`.
            if (t.k == 0) tile_u = carried(tile_f, carry, tile_u), tile_f = 0;
            publish(entries + t.k * CL * W + tid * W, tile_f, tile_u);
            fold_entries(entries + first * CL * W, tid * W, CL * W, static_cast<uint32_t>(t.k - first), group_f, group_u);
            if (t.k + 1 == first + s.p.group) publish(groups + g * CL * W + tid * W, group_f * tile_f, carried(tile_f, group_u, tile_u));
        } else if (tid >= CL && tid < 2 * CL && t.c0 + tid - CL < t.c1) {
            // The groups before this one, from the first one's constant on.
            C any = 1, state = 0;
            fold_entries(groups, (tid - CL) * W, CL * W, static_cast<uint32_t>(g), any, state);
            before_group[tid - CL] = state;
        }
        __syncthreads();
        if (folds && t.k > 0) carry = g == 0 ? group_u : (t.k == first ? before_group[tid] : carried(group_f, before_group[tid], group_u));
    }
    if (folds) {
        constexpr int kAhead = 8;
        for (int i0 = 0; i0 < P; i0 += kAhead) {
            C nf[kAhead], nu[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; ++i) nf[i] = part_f(i0 + i), nu[i] = part_u(i0 + i);
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                part_u(i0 + i) = carry;
                carry = carried(nf[i], carry, nu[i]);
            }
        }
        if (t.k + 1 == s.p.tiles && a.exit.p != nullptr) store_state<T>(a.exit.p, a.exit.at(t.b, cj), a.exit.wide, carry);
    }
    __syncthreads();
    if constexpr (RP > 1) {
        if (has_run) {
            C into = run_u[run][run_channel];
#pragma unroll
            for (int i = 0; i < RP; ++i) {
                const C nf = slot_f[run * RP + i][run_channel], nu = slot_u[run * RP + i][run_channel];
                slot_u[run * RP + i][run_channel] = into;
                into = carried(nf, into, nu);
            }
        }
        __syncthreads();
    }
    C e[V];
#pragma unroll
    for (int j = 0; j < V; ++j) e[j] = t.lane_on ? slot_u[r][t.at + j] : C(0);
    if (t.lane_on) {
        const bool wide_gate = BACK && sizeof(T) < sizeof(C) && a.d_gate_wide;
        char *const to = base_of(t, BACK ? a.d_gate : a.out, 0, wide_gate ? sizeof(C) : sizeof(T));
        char *const to_input = BACK ? base(t, a.d_input) : nullptr;
#pragma unroll
        for (int i = 0; i < S; ++i) {
            Vec<T, V> out;
            if constexpr (!BACK) {
                C y[V];
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    C f, add;
                    map(i, j, f, add);
                    y[j] = e[j] = fma_(f, e[j], add);
                }
                out.round(y);
                out.only(t.has(i));
                if (i < t.end) out.template store<kStorePast>(row(to, t, a.out, i));
            } else {
                C dg[V], dx[V];
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    C before = now.before[i].get(j);
                    if (i == t.first && a.initial.p != nullptr) {
                        before = load_state<T>(a.initial.p, a.initial.at(t.b, t.c0 + t.at + j), a.initial.wide);
                    }
                    const C g = now.grad[i].get(j) + e[j];
                    C x = 0;
                    if constexpr (FORM == HMN_GATE_SIGMOID) x = now.input[i].get(j);
                    e[j] = step_back<T, FORM>(now.gate[i].get(j), x, g, before, dg[j], dx[j]);
                }
                if (wide_gate) {
                    Vec<C, V> wide;
                    wide.round(dg);
                    wide.only(t.has(i));
                    if (i < t.end) wide.template store<kStorePast>(reinterpret_cast<C *>(row_of(to, t, a.d_gate, i, sizeof(C))));
                } else {
                    out.round(dg);
                    out.only(t.has(i));
                    if (i < t.end) out.template store<kStorePast>(row(to, t, a.d_gate, i));
                }
                out.round(dx);
                out.only(t.has(i));
                if (i < t.end) out.template store<kStorePast>(row(to_input, t, a.d_input, i));
            }
        }
    }
}

// The shapes in use. Lanes hold 16 bytes of channels where channels lie next to each other, else one; sequences that one
// short tile covers take that. Backwards a lane has four operands in registers, and more slots of fewer steps keep two
// workgroups on a compute unit ([4, 4096, 2048] bf16: 97 us, 113 with the forward shape; forwards [8, 2048, 4096] 86 us,
// 88 with the backward one).
template <class T>
constexpr int kVector = 16 / static_cast<int>(sizeof(T));
constexpr int kSlots = 16, kShortest = kSlots * 1;
template <class T>
using ShortShape = ScanShape<T, kVector<T>, kSlots, 1>;
template <class T, bool BACK>
using LongShape = ScanShape<T, kVector<T>, BACK ? 32 : 16, BACK ? 4 : 6>;
// Of few vectors of channels: the lanes that those would leave idle go along the sequence ([240, 8324, 8] f32 101 us, 450
// with the long shape; [75, 906, 39] bf16 19 and 37). Of up to four blocks of channels (two backwards) too, where the long
// shape would need several tiles ([240, 8324, 128] bf16 504 us and 637; backwards, 64 channels, 415 and 542, but 128
// channels 799 and 662).
template <class T>
using NarrowShape = ScanShape<T, kVector<T>, 128, 4>;
template <class T, bool BACK>
bool narrow(const RecurrenceArgs &a) {
    constexpr int64_t kOfBlock = NarrowShape<T>::kChannels;
    return a.C <= kOfBlock || (a.T > LongShape<T, BACK>::kSteps && a.C <= (BACK ? 2 : 4) * kOfBlock);
}
template <class T>
using LoneShape = ScanShape<T, 1, kSlots, 8>;
// Of up to eight channels in all, whatever their places: longer tiles ([64, 12964, 2] bf16 40 us, 175 with the lone shape).
template <class T>
using FewShape = ScanShape<T, 1, 64, 8>;

// Queues a scan of this shape.
template <class Shape, class T, int FORM, bool BACK, int PASSING>
void launch_scan(hipStream_t stream, const RecurrenceArgs &a, void *room) {
    ScanArgs s{a, Shape::plan(a.T, a.C), static_cast<uint64_t *>(room)};
    const uint32_t tiles = static_cast<uint32_t>(a.B * s.p.blocks * s.p.tiles);
    if (Shape::kSteps == kShortest || s.p.tiles <= 1) {
        scan_kernel<T, Shape, FORM, BACK, false, PASSING><<<tiles, kScanBlock, 0, stream>>>(s);
        return;
    }
    if constexpr (Shape::kSteps > kShortest) {
        const int64_t words = Shape::words(s.p, a.B), clearing = (words + 4 * kBlock - 1) / (4 * kBlock);
        scan_clear_kernel<<<static_cast<uint32_t>(clearing < 2048 ? clearing : 2048), kBlock, 0, stream>>>(s.room, words);
        scan_kernel<T, Shape, FORM, BACK, true, PASSING><<<tiles, kScanBlock, 0, stream>>>(s);
    }
}

// Calls f(shape) for every shape that the operands' strides and the direction may call for.
template <class T, class F>
void with_scan_shapes(int64_t steps, F &&f) {
    if (steps <= kShortest) {
        f(ShortShape<T>{});
    } else {
        f(LongShape<T, false>{});
        f(LongShape<T, true>{});
        f(NarrowShape<T>{});
    }
    f(LoneShape<T>{});
    f(FewShape<T>{});
}

template <bool BACK>
void queue_scan(hipStream_t stream, int32_t dtype, int32_t form, const RecurrenceArgs &a, const ScanLayout &layout, void *room) {
    with_float_type(dtype, [&](auto tag) {
        using T = typename decltype(tag)::type;
        with_code(form, std::integer_sequence<int, HMN_GATE_FACTOR, HMN_GATE_SIGMOID>{}, [&](auto f) {
            constexpr int FORM = decltype(f)::value;
            if (a.C <= FewShape<T>::kChannels && (!layout.adjacent || a.C < kVector<T>)) {
                launch_scan<FewShape<T>, T, FORM, BACK, kThroughCaches>(stream, a, room);
            } else if (!layout.adjacent || a.C < kVector<T>) {
                launch_scan<LoneShape<T>, T, FORM, BACK, kThroughCaches>(stream, a, room);
            } else if (a.T <= kShortest) {
                launch_scan<ShortShape<T>, T, FORM, BACK, kThroughCaches>(stream, a, room);
            } else if (narrow<T, BACK>(a)) {
                launch_scan<NarrowShape<T>, T, FORM, BACK, kThroughCaches>(stream, a, room);
            } else {
                constexpr int64_t kOperands = BACK ? (FORM == HMN_GATE_SIGMOID ? 6 : 5) : 3;
                const int64_t bytes = a.B * a.T * a.C * kOperands * static_cast<int64_t>(sizeof(T));
                with_passing(passing(bytes, layout.whole_lines), [&](auto p) {
                    launch_scan<LongShape<T, BACK>, T, FORM, BACK, decltype(p)::value>(stream, a, room);
                });
            }
        });
    });
}

}  // namespace nn
}  // namespace hmr
