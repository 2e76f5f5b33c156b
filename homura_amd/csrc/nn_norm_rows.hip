// Group normalisation of groups that fit a wave's or a workgroup's registers, and the sum of the weights' gradients.
#include "nn_norm.hpp"

namespace hmr {
namespace nn {
namespace {

constexpr int kWaves = kBlock / 64;

struct RowsArgs {
    NormArgs a;
    RowsPlan p;
    int32_t activation;
    bool weights;   // backwards: whether the weights' gradients are wanted,
    void *partial;  // and room for [2][walkers][C] sums in the computation type
};

// Where a lane's vectors lie, the same for every row it visits.
template <int M>
struct LaneVectors {
    bool on[M];
    int64_t src[M], out[M], grad[M];  // offsets from the row's first channel
    int64_t channel[M];
};

template <class T, int V, int M, bool WIDE, bool PAST, bool BACK>
__global__ void __launch_bounds__(kBlock) rows_kernel(RowsArgs s) {
    using C = typename Comp<T>::C;
    const NormArgs &a = s.a;
    const RowsPlan &p = s.p;
    // Rows a lane works on at a time.
    constexpr int U = !BACK && M == 1 ? 2 : 1;
    constexpr bool kKeep = M * V <= 16;  // the weights in registers
    const int tid = threadIdx.x, wave = tid >> 6, lane = WIDE ? tid : tid & 63;
    const int64_t block = blockIdx.x % p.blocks, walker = blockIdx.x / p.blocks;
    const int slot = lane / p.lanes, first = lane % p.lanes;
    const int side = WIDE ? 1 : static_cast<int>(64 / p.lanes / p.rows);  // groups side by side of one row
    const int row = slot / side;                                          // of the wave's rows
    const int64_t g = block * side + slot % side;
    const bool slot_on = row < p.rows && g < a.G;
    LaneVectors<M> at;
#pragma unroll
    for (int m = 0; m < M; ++m) {
        const int j = first + m * p.lanes;
        const int position = j / p.per_position, in = (j - position * p.per_position) * V;
        at.on[m] = slot_on && j < p.vectors;
        at.channel[m] = at.on[m] ? g * a.W + in : 0;
        at.src[m] = position * a.src.ss + at.channel[m], at.out[m] = position * a.out.ss + at.channel[m];
        at.grad[m] = BACK ? position * a.grad.ss + at.channel[m] : 0;
    }
    // Backwards a vector without elements has weights and biases of zero: those of channel 0, which it would load, may be
    // anything, and what it computes is added to its group's sums.
    auto fetch_weights = [&](int m, C(&w)[V], C(&b)[V]) {
        load_channels<T, V>(a.weight, at.channel[m], C(1), w);
        load_channels<T, V>(a.bias, at.channel[m], C(0), b);
        if constexpr (BACK) {
#pragma unroll
            for (int i = 0; i < V; ++i) w[i] = at.on[m] ? w[i] : C(0), b[i] = at.on[m] ? b[i] : C(0);
        }
    };
    C keep_w[kKeep ? M : 1][V], keep_b[kKeep ? M : 1][V];
    if constexpr (kKeep) {
#pragma unroll
        for (int m = 0; m < M; ++m) fetch_weights(m, keep_w[m], keep_b[m]);
    }
    // The sums of both over a group's lanes: moments in f64, the gradient's two sums in the computation type (V additions in a
    // row for each of a lane's M vectors, then those and the lanes pairwise or nearly so: in f32 as good as a pairwise sum, and
    // in f64 [8192, 4096] f16 took 55 us for 52).
    using A = std::conditional_t<BACK, C, double>;
    __shared__ A wide_sums[2][kWaves];
    auto group_sums = [&](A &x, A &y) {
        if constexpr (!WIDE) {
            x = lanes_sum(x, p.lanes), y = lanes_sum(y, p.lanes);
        } else {
            x = lanes_sum(x, 64), y = lanes_sum(y, 64);
            __syncthreads();
            if ((tid & 63) == 0) wide_sums[0][wave] = x, wide_sums[1][wave] = y;
            __syncthreads();
            x = y = 0;
#pragma unroll
            for (int k = 0; k < kWaves; ++k) x += wide_sums[0][k], y += wide_sums[1][k];
        }
    };
    // Many vectors are worked on one after the other: the scheduler would hold all their intermediate values at once.
    auto one_by_one = [] {
        if constexpr (M > 2) __builtin_amdgcn_sched_barrier(0);
    };
    const double share = 1.0 / (static_cast<double>(a.S) * static_cast<double>(a.W));
    // The lane's sums of d and d * hat over its rows, in f32 by runs.
    constexpr bool kRuns = BACK && sizeof(C) == 4;
    C sum_d[BACK ? M : 1][V], sum_dh[BACK ? M : 1][V], all_d[kRuns ? M : 1][V], all_dh[kRuns ? M : 1][V];
    int run = 0;
    if constexpr (BACK) {
#pragma unroll
        for (int m = 0; m < M; ++m) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                sum_d[m][i] = sum_dh[m][i] = 0;
                if constexpr (kRuns) all_d[m][i] = all_dh[m][i] = 0;
            }
        }
    }
    auto end_run = [&] {
        run = 0;
#pragma unroll
        for (int m = 0; m < (kRuns ? M : 0); ++m) {
#pragma unroll
            for (int i = 0; i < V; ++i) add_run(all_d[m][i], sum_d[m][i]), add_run(all_dh[m][i], sum_dh[m][i]);
        }
    };
    // The next rows are under way while these are worked on.
    struct Rows {
        Vec<T, V> x[U][M], dy[BACK ? U : 1][M];
        C mean[U], rstd[U];  // backwards
        bool on[U];
    };
    auto fetch = [&](int64_t n0, Rows &rows) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t n = n0 + u * p.rows + row;
            rows.on[u] = n < a.N;
            if constexpr (BACK) {
                rows.mean[u] = rows.rstd[u] = 0;
                if (rows.on[u] && slot_on) {
                    rows.mean[u] = reinterpret_cast<const C *>(a.mean.p)[a.mean.at(n, g)];
                    rows.rstd[u] = reinterpret_cast<const C *>(a.rstd.p)[a.rstd.at(n, g)];
                }
            }
#pragma unroll
            for (int m = 0; m < M; ++m) {
                rows.x[u][m].only(false);
                if constexpr (BACK) rows.dy[u][m].only(false);
                if (rows.on[u] && at.on[m]) {
                    rows.x[u][m].template load<PAST>(reinterpret_cast<const T *>(a.src.p) + n * a.src.sn + at.src[m]);
                    if constexpr (BACK) rows.dy[u][m].template load<PAST>(reinterpret_cast<const T *>(a.grad.p) + n * a.grad.sn + at.grad[m]);
                }
            }
        }
    };
    const int64_t stride = p.walkers * (WIDE ? 1 : kWaves) * U * p.rows;
    int64_t n0 = (walker * (WIDE ? 1 : kWaves) + (WIDE ? 0 : wave)) * U * p.rows;
    Rows next;
    fetch(n0, next);
    for (; n0 < a.N; n0 += stride) {
        Rows now = next;
        auto &x = now.x;
        fetch(n0 + stride, next);
        int64_t n[U];
#pragma unroll
        for (int u = 0; u < U; ++u) n[u] = n0 + u * p.rows + row;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            auto weights = [&](int m, C(&w)[V], C(&b)[V]) {
                if constexpr (kKeep) {
#pragma unroll
                    for (int i = 0; i < V; ++i) w[i] = keep_w[m][i], b[i] = keep_b[m][i];
                } else {
                    fetch_weights(m, w, b);
                }
            };
            if constexpr (!BACK) {
                // Lanes without elements hold zeros. In f64 the squares of 16- and 32-bit elements are exact, and the variance
                // from their sum is off by some 2^-53 (mean / deviation)^2 of itself and the additions' share: up to 2^10
                // deviations less than f32 holds. Groups farther out, as F64 ones always, sum squares about the mean too.
                double sum = 0, squares = 0;
#pragma unroll
                for (int m = 0; m < M; ++m) {
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        const double v = x[u][m].get(i);
                        sum += v;
                        if constexpr (!std::is_same_v<T, double>) squares = __builtin_fma(v, v, squares);
                    }
                    one_by_one();
                }
                group_sums(sum, squares);
                const double mean = sum * share;
                double variance;
                auto about_the_mean = [&] {
                    double centred = 0, none = 0;
#pragma unroll
                    for (int m = 0; m < M; ++m) {
#pragma unroll
                        for (int i = 0; i < V; ++i) {
                            const double v = x[u][m].get(i) - mean;
                            if (at.on[m]) centred = __builtin_fma(v, v, centred);
                        }
                        one_by_one();
                    }
                    group_sums(centred, none);
                    return centred * share;
                };
                if constexpr (std::is_same_v<T, double>) {
                    variance = about_the_mean();
                } else {
                    variance = __builtin_fma(-mean, mean, squares * share);
                    // Each group by its own mean and variance, whatever else the wave holds (a wide one is the workgroup's).
                    const bool far = mean * mean > 0x1p20 * variance;
                    if (__any(far)) {
                        const double centred = about_the_mean();
                        variance = far ? centred : variance;
                    }
                }
                const double rstd = reciprocal_root(variance + a.eps);
                if (now.on[u] && slot_on && first == 0) {
                    if (a.mean.p != nullptr) reinterpret_cast<C *>(a.mean.p)[a.mean.at(n[u], g)] = static_cast<C>(mean);
                    if (a.rstd.p != nullptr) reinterpret_cast<C *>(a.rstd.p)[a.rstd.at(n[u], g)] = static_cast<C>(rstd);
                }
                if constexpr (M > 2) {
#pragma unroll
                    for (int m = 0; m < M; ++m) x[u][m].forget();
                }
                const Centre<C> centre(mean, rstd);
#pragma unroll
                for (int m = 0; m < M; ++m) {
                    C w[V], b[V], z[V];
                    weights(m, w, b);
#pragma unroll
                    for (int i = 0; i < V; ++i) z[i] = fma_(centre.hat(x[u][m].get(i)), w[i], b[i]);
                    activate_all<T, V>(s.activation, z);
                    Vec<T, V> y;
                    y.round(z);
                    if (now.on[u] && at.on[m]) y.template store<PAST>(reinterpret_cast<T *>(a.out.p) + n[u] * a.out.sn + at.out[m]);
                    one_by_one();
                }
            } else {
                const C rstd = now.rstd[u];
                C hat[M][V], wd[M][V];
                C wd_sum = 0, wdh_sum = 0;
                // A row that is not there adds nothing, whatever its channels' weights would make of zeros; nor does a
                // vector without elements: its elements, mean, weights and gradients are zero.
                if (!now.on[u]) {
#pragma unroll
                    for (int m = 0; m < M; ++m) {
#pragma unroll
                        for (int i = 0; i < V; ++i) hat[m][i] = wd[m][i] = 0;
                    }
                } else {
#pragma unroll
                    for (int m = 0; m < M; ++m) {
                        C w[V], b[V], z[V];
                        weights(m, w, b);
                        const C mean = at.on[m] ? now.mean[u] : C(0);
#pragma unroll
                        for (int i = 0; i < V; ++i) {
                            hat[m][i] = (x[u][m].get(i) - mean) * rstd;
                            z[i] = fma_(hat[m][i], w[i], b[i]);
                        }
                        slope_all<T, V>(s.activation, z);
                        C part = 0, part_h = 0;
#pragma unroll
                        for (int i = 0; i < V; ++i) {
                            const C d = now.dy[u][m].get(i) * z[i];  // a lane without elements has zero gradients
                            sum_d[m][i] += d, sum_dh[m][i] = fma_(d, hat[m][i], sum_dh[m][i]);
                            wd[m][i] = w[i] * d;
                            part += wd[m][i], part_h = fma_(wd[m][i], hat[m][i], part_h);
                        }
                        wd_sum += part, wdh_sum += part_h;
                        one_by_one();
                    }
                }
                group_sums(wd_sum, wdh_sum);
                const C d_mean = wd_sum * static_cast<C>(share), dh_mean = wdh_sum * static_cast<C>(share);
#pragma unroll
                for (int m = 0; m < M; ++m) {
                    C r[V];
#pragma unroll
                    for (int i = 0; i < V; ++i) r[i] = rstd * fma_(-hat[m][i], dh_mean, wd[m][i] - d_mean);
                    Vec<T, V> dx;
                    dx.round(r);
                    if (now.on[u] && at.on[m]) dx.template store<PAST>(reinterpret_cast<T *>(a.out.p) + n[u] * a.out.sn + at.out[m]);
                }
            }
        }
        if constexpr (kRuns) {
            if (++run == kMostRun) end_run();
        }
    }
    if constexpr (BACK) {
        if (!s.weights) return;
        if constexpr (kRuns) {
#pragma unroll
            for (int m = 0; m < M; ++m) {
#pragma unroll
                for (int i = 0; i < V; ++i) sum_d[m][i] += all_d[m][i], sum_dh[m][i] += all_dh[m][i];
            }
        }
        // The lanes of one channel (a lane of every wave; of several positions and rows where those are side by side) are
        // added in order by the thread that owns the channel in the workgroup's block.
        constexpr int kSpread = WIDE ? kBlock : 64;
        extern __shared__ char sums_raw[];
        C *sums = reinterpret_cast<C *>(sums_raw);  // [waves][M][lanes][V]
        C *partial = static_cast<C *>(s.partial);
        const int64_t c0 = block * side * a.W;
        const int64_t channels = (c0 + side * a.W < a.C ? c0 + side * a.W : a.C) - c0;
        const int positions = static_cast<int>(a.S);
        __shared__ double parts[kBlock];
        // A lone walker's sums are the gradients.
        auto put = [&](int which, int64_t c, double total) {
            const PerChannel &to = which == 0 ? a.d_weight : a.d_bias;
            if (p.walkers > 1) partial[(which * p.walkers + walker) * a.C + c] = static_cast<C>(total);
            else if (to.p != nullptr) store_state<T>(to.p, c * to.sc, to.wide, static_cast<C>(total));
        };
        for (int which = 0; which < 2; ++which) {
            __syncthreads();
#pragma unroll
            for (int m = 0; m < M; ++m) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    sums[((static_cast<int64_t>(WIDE ? 0 : wave) * M + m) * kSpread + lane) * V + i] = which == 0 ? sum_dh[m][i] : sum_d[m][i];
                }
            }
            __syncthreads();
            // `share` threads a channel where there are fewer channels than threads.
            const int entries = (WIDE ? 1 : kWaves) * p.rows * positions;
            const int share = channels < kBlock && entries != kWaves ? kBlock / static_cast<int>(channels) : 1;
            for (int64_t k = tid; k < channels * share; k += kBlock) {
                const int c = static_cast<int>(k % channels), group = static_cast<int>(c / a.W), in = static_cast<int>(c - group * a.W);
                double total = 0;
                auto add = [&](int w, int r, int position) {
                    const int j = position * p.per_position + in / V;
                    const int l = (r * side + group) * p.lanes + j % p.lanes, m = j / p.lanes;
                    total += sums[((w * M + m) * kSpread + l) * V + in % V];
                };
                if (entries == kWaves) {  // a position and a row a wave: the usual tokens
#pragma unroll
                    for (int w = 0; w < kWaves; ++w) add(w, 0, 0);
                } else {
                    for (int e = static_cast<int>(k / channels); e < entries; e += share) add(e / positions / p.rows, e / positions % p.rows, e % positions);
                }
                if (share == 1) put(which, c0 + c, total);
                else parts[k] = total;
            }
            if (share > 1) {
                __syncthreads();
                if (tid < channels) {
                    double total = 0;
                    for (int k = 0; k < share; ++k) total += parts[tid + k * channels];
                    put(which, c0 + tid, total);
                }
            }
        }
    }
}

// ---- the weights' gradients ---------------------------------------------------------------------------------------------
//
template <class T>
__global__ void __launch_bounds__(kBlock) weights_sum_kernel(NormArgs a, const typename Comp<T>::C *partial, int64_t parts) {
    sum_channels<T>(a, partial, parts, blockIdx.x);
}

int power_of_two(int64_t at_least) {
    int p = 1;
    while (p < at_least) p *= 2;
    return p;
}

template <class T, int V, bool BACK>
void launch_rows(hipStream_t stream, const RowsArgs &s, bool past) {
    using C = typename Comp<T>::C;
    const uint32_t groups = static_cast<uint32_t>(s.p.blocks * s.p.walkers);
    auto run = [&](auto m, auto wide, auto passing) {
        constexpr int M = decltype(m)::value;
        constexpr bool WIDE = decltype(wide)::value != 0, PAST = decltype(passing)::value != 0;
        const size_t lds = BACK ? static_cast<size_t>(kBlock) * M * V * sizeof(C) : 0;
        rows_kernel<T, V, M, WIDE, PAST, BACK><<<groups, kBlock, lds, stream>>>(s);
    };
    auto pass = [&](auto m, auto wide) {
        if constexpr (V * sizeof(T) == 16) {
            if (past) return run(m, wide, IntTag<1>{});
        }
        run(m, wide, IntTag<0>{});
    };
    if (s.p.wide) {
        if (s.p.m == 2) pass(IntTag<2>{}, IntTag<1>{});
        else pass(IntTag<4>{}, IntTag<1>{});
    } else {
        switch (s.p.m) {
            case 1: pass(IntTag<1>{}, IntTag<0>{}); break;
            case 2: pass(IntTag<2>{}, IntTag<0>{}); break;
            case 4: pass(IntTag<4>{}, IntTag<0>{}); break;
            default:
                if constexpr (!BACK) pass(IntTag<8>{}, IntTag<0>{});
        }
    }
}

template <class T, bool BACK>
void launch_width(hipStream_t stream, const RowsArgs &s, bool past) {
    constexpr int kFull = 16 / static_cast<int>(sizeof(T));
    if (s.p.v == kFull) return launch_rows<T, kFull, BACK>(stream, s, past);
    if constexpr (kFull == 8) {
        if (s.p.v == 2) return launch_rows<T, 2, BACK>(stream, s, past);
    }
    launch_rows<T, 1, BACK>(stream, s, past);
}

}  // namespace

RowsPlan rows_plan(const NormArgs &a, int32_t dtype, bool backward) {
    RowsPlan p{};
    const int full = 16 / dtype_size(dtype);
    p.v = a.W % full == 0 ? full : (full == 8 && a.W % 2 == 0 ? 2 : 1);
    // Of maps only small ones: a group's channels at one position are short runs of memory (and, backwards, a channel's sum
    // meets every position of it at the end).
    if (a.S == 0 || a.W == 0 || a.S > 64 || a.W > 65536) return p;
    p.per_position = static_cast<int32_t>(a.W / p.v);
    const int64_t vectors = a.S * p.per_position;
    const int most = backward ? 4 : 8;  // vectors of a lane
    if (vectors <= 64 * most) {
        p.lanes = vectors < 64 ? power_of_two(vectors) : 64;
        p.m = power_of_two((vectors + p.lanes - 1) / p.lanes);
    } else if (a.S == 1 && vectors <= kBlock * 4) {
        p.wide = true, p.lanes = kBlock;
        p.m = vectors <= kBlock * 2 ? 2 : 4;
    } else {
        return p;
    }
    p.vectors = static_cast<int32_t>(vectors);
    const int64_t slots = p.wide ? 1 : 64 / p.lanes;
    p.rows = a.G < slots ? static_cast<int32_t>(slots / a.G) : 1;
    const int64_t side = slots / p.rows;  // groups of one row in a wave (as the kernel counts them)
    p.blocks = (a.G + side - 1) / side;
    // Enough workgroups to fill the chip four times over forwards; backwards each leaves a row of partial sums, so as many as
    // keep it busy once with four on a compute unit.
    const int64_t target = backward ? 1024 : 4096, rows_at_once = (p.wide ? 1 : kWaves) * p.rows;
    int64_t walkers = (target + p.blocks - 1) / p.blocks;
    const int64_t useful = (a.N + rows_at_once - 1) / rows_at_once;
    p.walkers = walkers < useful ? walkers : (useful > 0 ? useful : 1);
    if (!fits_launch(p.blocks * p.walkers, kBlock)) p.m = 0;
    return p;
}

int64_t norm_rows_room(const NormArgs &a, int32_t dtype, bool backward) {
    if (!backward) return 0;
    const RowsPlan p = rows_plan(a, dtype, true);
    return p.m == 0 ? 0 : 2 * p.walkers * a.C * dtype_size(wide_type(dtype));
}

bool queue_norm_rows(hipStream_t stream, int32_t dtype, const NormArgs &a, int32_t activation, void *room, bool backward) {
    if (!channels_adjacent(a, backward)) return false;
    const bool weights = backward && (a.d_weight.p != nullptr || a.d_bias.p != nullptr);
    RowsArgs s{a, rows_plan(a, dtype, backward), activation, weights, room};
    if (s.p.m == 0 || a.N == 0) return false;
    const bool past = a.N * a.S * a.C * dtype_size(dtype) * (backward ? 3 : 2) > kCacheResidentBytes;
    with_float_type(dtype, [&](auto tag) {
        using T = typename decltype(tag)::type;
        if (backward) launch_width<T, true>(stream, s, past);
        else launch_width<T, false>(stream, s, past);
    });
    if (weights && s.p.walkers > 1) {
        with_float_type(dtype, [&](auto tag) {
            using T = typename decltype(tag)::type;
            weights_sum_kernel<T><<<static_cast<uint32_t>((a.C + kSumChannels - 1) / kSumChannels), kBlock, 0, stream>>>(
                a, static_cast<const typename Comp<T>::C *>(room), s.p.walkers);
        });
    }
    return true;
}

}  // namespace nn
}  // namespace hmr
