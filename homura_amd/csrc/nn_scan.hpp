// The scan's kernels (nn_recurrence.hpp says how a tile gets the value that enters it).
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

// Folds `count` published entries, `apart` words from each other, in order, onto (f, u).
template <class C>
__device__ __forceinline__ void fold_entries(const uint64_t *p, int64_t apart, int64_t count, C &f, C &u) {
    constexpr int kAhead = 8, W = sizeof(C) / 4;
    for (int64_t i = 0; i < count; i += kAhead) {
        uint64_t w[kAhead][W];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const uint64_t *q = p + (i + j < count ? i + j : count - 1) * apart;
#pragma unroll
            for (int k = 0; k < W; ++k) w[j][k] = peek(q + k);
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            if (i + j < count) {
                const uint64_t *q = p + (i + j) * apart;
                C ef, eu;
                if constexpr (W == 1) {
                    const uint64_t x = await(q, w[j][0]);
                    ef = bits_as<float>(static_cast<uint32_t>(x)), eu = bits_as<float>(static_cast<uint32_t>(x >> 32));
                } else {
                    ef = bits_as<double>(await(q, w[j][0])), eu = bits_as<double>(await(q + 1, w[j][1]));
                }
                u = carried(ef, u, eu);
                f *= ef;
            }
        }
    }
}

template <class T, int V, int R, int S, int FORM, bool BACK, bool CHAIN>
__global__ void __launch_bounds__(kScanBlock) scan_kernel(ScanArgs s) {
    using C = typename Comp<T>::C;
    using Shape = ScanShape<T, V, R, S>;
    constexpr int L = Shape::kLanes, CL = Shape::kChannels, TT = Shape::kSteps, W = Shape::kWords;
    constexpr int kBuffers = CHAIN ? 1 : 2;  // a walk's next tile writes the other pair of buffers
    static_assert(TT <= kMostSteps && CL <= kMostChannels, "spans the host checks for");
    static_assert(CL <= kScanBlock && (!CHAIN || 2 * CL <= kScanBlock), "a thread per channel folds slots");
    __shared__ C slot_f[kBuffers][R][CL], slot_u[kBuffers][R][CL];
    __shared__ C before_group[CHAIN ? CL : 1];
    __shared__ uint32_t ticket_here;
    const RecurrenceArgs &a = s.a;
    const int tid = threadIdx.x, l = tid % L, r = tid / L;
    int64_t chain = blockIdx.x, k0 = 0, k1 = s.p.tiles;
    if constexpr (CHAIN) {
        if (tid == 0) ticket_here = atomicAdd(reinterpret_cast<uint32_t *>(s.room), 1u);
        __syncthreads();
        const uint32_t ticket = __builtin_amdgcn_readfirstlane(ticket_here);
        k0 = ticket / s.p.chains, chain = ticket % s.p.chains, k1 = k0 + 1;
    }
    const int64_t b = chain / s.p.blocks, steps = a.steps(b);
    // A vector never crosses the last channel: the last block begins early enough to have one, the last lane's moves back
    // over its neighbour's channels, and both compute the same for those.
    const int64_t block0 = (chain % s.p.blocks) * CL;
    const int64_t c0 = V > 1 && block0 > a.C - V ? a.C - V : block0;
    const bool lane_on = c0 + l * V < a.C;
    const int64_t c = V > 1 && c0 + l * V > a.C - V ? a.C - V : c0 + l * V;
    const int at = static_cast<int>(c - c0);  // the lane's first channel inside the block
    const int64_t cj = c0 + tid;              // the channel whose slots this thread folds
    const bool folds = tid < CL && cj < a.C;

    struct Raw {
        Vec<T, V> gate[S], input[S], grad[BACK ? S : 1], before[BACK ? S : 1];
    };
    // The lane's steps of tile k: those from `from` to `to` lie inside the sequence, those from `end` on past the batch's
    // last; `first` is the sequence's first step (if it is the lane's at all), which backwards starts from `initial`.
    struct Span {
        int from, to, end, first;
        __device__ __forceinline__ bool has(int i) const { return i >= from && i < to; }
    };
    auto clamped = [](int64_t n) { return static_cast<int>(n < 0 ? 0 : (n > S ? S : n)); };
    auto span_of = [&](int64_t k) {
        const int64_t q0 = k * TT + r * S;
        const int end = clamped(a.T - q0);
        if constexpr (BACK) return Span{clamped(a.T - steps - q0), end, end, a.T - q0 <= S ? static_cast<int>(a.T - 1 - q0) : S};
        else return Span{0, clamped(steps - q0), end, S};
    };
    // Where a tile lies: the address of its earliest step (less `back`) and first channel, the same for the whole
    // workgroup, and the lane's offset from there in 32 bits (the host has checked that a tile spans less).
    auto base = [&](const Sequences &x, int64_t k, int back = 0) {
        const int64_t first = BACK ? a.T - (k + 1) * TT : k * TT;
        return x.p + (b * x.sb + (first - back) * x.st + c0 * x.sc) * static_cast<int64_t>(sizeof(T));
    };
    auto row = [&](char *from, const Sequences &x, int i) {
        const int step = BACK ? TT - 1 - (r * S + i) : r * S + i;
        const uint32_t off = (static_cast<uint32_t>(step) * static_cast<uint32_t>(x.st) + static_cast<uint32_t>(at) * static_cast<uint32_t>(x.sc)) *
                             static_cast<uint32_t>(sizeof(T));
        return reinterpret_cast<T *>(from + off);
    };
    // Steps outside the sequence get what maps a value to itself: a factor of one (sigmoid's at infinity) and nothing to add.
    auto load = [&](int64_t k, Raw &raw) {
        const Span span = span_of(k);
        char *gate = base(a.gate, k), *input = nullptr, *grad = nullptr, *before = nullptr;
        if constexpr (!BACK || FORM == HMN_GATE_SIGMOID) input = base(a.input, k);
        if constexpr (BACK) grad = base(a.grad, k), before = base(a.state, k, 1);
#pragma unroll
        for (int i = 0; i < S; ++i) {
            raw.gate[i].fill(FORM == HMN_GATE_FACTOR ? C(1) : C(__builtin_inf()));
            raw.input[i].fill(C(0));
            if constexpr (BACK) raw.grad[i].fill(C(0)), raw.before[i].fill(C(0));
            if (lane_on && span.has(i)) {
                raw.gate[i].load(row(gate, a.gate, i));
                if constexpr (!BACK || FORM == HMN_GATE_SIGMOID) raw.input[i].load(row(input, a.input, i));
                if constexpr (BACK) {
                    raw.grad[i].load(row(grad, a.grad, i));
                    if (i != span.first) raw.before[i].load(row(before, a.state, i));
                }
            }
        }
    };
    C carry = 0;  // of channel cj: the value that enters the tile, then the one that leaves it
    if (folds && (!CHAIN || k0 == 0) && a.entry.p != nullptr) carry = load_state<T>(a.entry.p, a.entry.at(b, cj), a.entry.wide);

    // Whether the maps are computed again when the steps are run rather than kept: where that costs next to nothing.
    constexpr bool kAgain = BACK || FORM == HMN_GATE_FACTOR;
    auto work = [&](int64_t k, Raw &raw, int buffer) {
        const Span span = span_of(k);
        // The lane's steps as maps, and their fold.
        C kept_f[kAgain ? 1 : S][V], kept_u[kAgain ? 1 : S][V], fold_f[V], fold_u[V];
        auto map = [&](int i, int j, C &f, C &u) {
            const C z = raw.gate[i].get(j);
            if constexpr (!BACK) {
                factor_and_input<FORM>(z, raw.input[i].get(j), f, u);
            } else {
                C rest;
                if constexpr (FORM == HMN_GATE_SIGMOID) sigmoid_pair(z, f, rest);
                else f = z;
                u = f * raw.grad[i].get(j);
            }
        };
#pragma unroll
        for (int i = 0; i < S; ++i) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                C f, u;
                map(i, j, f, u);
                fold_u[j] = i == 0 ? u : fma_(f, fold_u[j], u);
                fold_f[j] = i == 0 ? f : fold_f[j] * f;
                if constexpr (!kAgain) kept_f[i][j] = f, kept_u[i][j] = u;
            }
        }
        if constexpr (kAgain) {
#pragma unroll
            for (int i = 0; i < S; ++i) {
                raw.gate[i].forget();
                if constexpr (!BACK) raw.input[i].forget();
                else raw.grad[i].forget();
            }
        }
        if (lane_on) {
#pragma unroll
            for (int j = 0; j < V; ++j) slot_f[buffer][r][at + j] = fold_f[j], slot_u[buffer][r][at + j] = fold_u[j];
        }
        __syncthreads();
        if constexpr (CHAIN) {
            const int64_t g = k / s.p.group, first = g * s.p.group;
            uint64_t *entries = s.room + 8 + chain * s.p.tiles * CL * W;
            uint64_t *groups = s.room + 8 + (s.p.chains * s.p.tiles + chain * (s.p.tiles / s.p.group + 1)) * CL * W;
            C group_f = 1, group_u = 0;
            if (folds) {
                C tile_f = slot_f[0][0][tid], tile_u = slot_u[0][0][tid];
#pragma unroll 8
                for (int i = 1; i < R; ++i) {
                    const C nf = slot_f[0][i][tid];
                    tile_u = carried(nf, tile_u, slot_u[0][i][tid]);
                    tile_f *= nf;
                }
                // The first tile knows what enters it: its map is constant, and no other tile reads `entry`.
                if (k == 0) tile_u = carried(tile_f, carry, tile_u), tile_f = 0;
                publish(entries + (k * CL + tid) * W, tile_f, tile_u);
                fold_entries(entries + (first * CL + tid) * W, CL * W, k - first, group_f, group_u);
                if (k + 1 == first + s.p.group) publish(groups + (g * CL + tid) * W, group_f * tile_f, carried(tile_f, group_u, tile_u));
            } else if (tid >= CL && tid < 2 * CL && c0 + tid - CL < a.C) {
                // The groups before this one, from the first one's constant on.
                C any = 1, state = 0;
                fold_entries(groups + (tid - CL) * W, CL * W, g, any, state);
                before_group[tid - CL] = state;
            }
            __syncthreads();
            if (folds && k > 0) carry = g == 0 ? group_u : (k == first ? before_group[tid] : carried(group_f, before_group[tid], group_u));
        }
        if (folds) {
            constexpr int kAhead = 8;
            for (int i0 = 0; i0 < R; i0 += kAhead) {
                C nf[kAhead], nu[kAhead];
#pragma unroll
                for (int i = 0; i < kAhead; ++i) nf[i] = slot_f[buffer][i0 + i][tid], nu[i] = slot_u[buffer][i0 + i][tid];
#pragma unroll
                for (int i = 0; i < kAhead; ++i) {
                    slot_u[buffer][i0 + i][tid] = carry;
                    carry = carried(nf[i], carry, nu[i]);
                }
            }
        }
        __syncthreads();
        if (lane_on) {
            char *const to = base(BACK ? a.d_gate : a.out, k), *const to_input = BACK ? base(a.d_input, k) : nullptr;
            C e[V];
#pragma unroll
            for (int j = 0; j < V; ++j) e[j] = slot_u[buffer][r][at + j];
#pragma unroll
            for (int i = 0; i < S; ++i) {
                Vec<T, V> out;
                if constexpr (!BACK) {
                    C y[V];
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        C f, u;
                        if constexpr (kAgain) map(i, j, f, u);
                        else f = kept_f[i][j], u = kept_u[i][j];
                        y[j] = e[j] = fma_(f, e[j], u);
                    }
                    out.round(y);
                    out.only(span.has(i));
                    if (i < span.end) out.store(row(to, a.out, i));
                } else {
                    C dg[V], dx[V];
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        C before = raw.before[i].get(j);
                        if (i == span.first && a.initial.p != nullptr) before = load_state<T>(a.initial.p, a.initial.at(b, c + j), a.initial.wide);
                        const C g = raw.grad[i].get(j) + e[j];
                        C x = 0;
                        if constexpr (FORM == HMN_GATE_SIGMOID) x = raw.input[i].get(j);
                        e[j] = step_back<FORM>(raw.gate[i].get(j), x, g, before, dg[j], dx[j]);
                    }
                    out.round(dg);
                    out.only(span.has(i));
                    if (i < span.end) out.store(row(to, a.d_gate, i));
                    out.round(dx);
                    out.only(span.has(i));
                    if (i < span.end) out.store(row(to_input, a.d_input, i));
                }
            }
        }
    };

    Raw now;
    load(k0, now);
    for (int64_t k = k0; k < k1; ++k) {
        Raw next;
        if (!CHAIN && k + 1 < k1) load(k + 1, next);
        const int buffer = CHAIN ? 0 : static_cast<int>(k & 1);
        work(k, now, buffer);
        if (!CHAIN) now = next;
    }
    if (folds && k1 == s.p.tiles && a.exit.p != nullptr) store_state<T>(a.exit.p, a.exit.at(b, cj), a.exit.wide, carry);
}

// Queues a scan of this shape.
template <class T, int V, int R, int S, int FORM, bool BACK>
void launch_scan(hipStream_t stream, const RecurrenceArgs &a, void *room) {
    using Shape = ScanShape<T, V, R, S>;
    ScanArgs s{a, Shape::plan(a.B, a.T, a.C), static_cast<uint64_t *>(room)};
    if (s.p.walk) {
        scan_kernel<T, V, R, S, FORM, BACK, false><<<static_cast<uint32_t>(s.p.chains), kScanBlock, 0, stream>>>(s);
        return;
    }
    if constexpr (2 * Shape::kChannels <= kScanBlock) {
        const int64_t words = Shape::words(s.p), groups = (words + 4 * kBlock - 1) / (4 * kBlock);
        scan_clear_kernel<<<static_cast<uint32_t>(groups < 1024 ? groups : 1024), kBlock, 0, stream>>>(s.room, words);
        scan_kernel<T, V, R, S, FORM, BACK, true><<<static_cast<uint32_t>(s.p.chains * s.p.tiles), kScanBlock, 0, stream>>>(s);
    }
}

// The shapes in use. Lanes hold 16 bytes of channels where channels lie next to each other, else one.
template <class T>
constexpr int kVector = 16 / static_cast<int>(sizeof(T));
constexpr int kSlots = 16;
constexpr int kLongSteps = 8, kShortSteps = 2, kLoneSteps = 16;  // steps of a lane: long and short sequences; single channels

// Bytes of workspace for whichever shape the operands' strides will call for.
template <class T>
int64_t scan_room(int64_t B, int64_t steps, int64_t C) {
    auto words = [&](auto shape) { return decltype(shape)::words(decltype(shape)::plan(B, steps, C)); };
    int64_t most = words(ScanShape<T, kVector<T>, kSlots, kLongSteps>{});
    const int64_t lone = words(ScanShape<T, 1, kSlots, kLoneSteps>{});
    if (lone > most) most = lone;
    return 8 * most;
}

template <bool BACK>
void queue_scan(hipStream_t stream, int32_t dtype, int32_t form, const RecurrenceArgs &a, bool vectors, void *room) {
    with_float_type(dtype, [&](auto tag) {
        using T = typename decltype(tag)::type;
        with_code(form, std::integer_sequence<int, HMN_GATE_FACTOR, HMN_GATE_SIGMOID>{}, [&](auto f) {
            constexpr int FORM = decltype(f)::value;
            if (!vectors || a.C < kVector<T>) launch_scan<T, 1, kSlots, kLoneSteps, FORM, BACK>(stream, a, room);
            else if (a.T <= kSlots * kShortSteps) launch_scan<T, kVector<T>, kSlots, kShortSteps, FORM, BACK>(stream, a, room);
            else launch_scan<T, kVector<T>, kSlots, kLongSteps, FORM, BACK>(stream, a, room);
        });
    });
}

}  // namespace nn
}  // namespace hmr
