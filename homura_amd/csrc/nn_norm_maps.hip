// Group normalisation of groups that are spread over workgroups: chunks' sums, then the maps again.
#include "nn_norm.hpp"

namespace hmr {
namespace nn {
namespace {

// What is known of a set of a group's elements. 16-bit ones: in f64 the sum and the sum of squares, which are exact where
// their bits matter (elements within a few binades of a mean far from zero, up to 2^31 of them); the variance is their
// difference with the products' rounding errors. F32: the same sums of the elements less the group's first one, from which
// the mean of m elements is at most sqrt(m) deviations away, so that the variance is off by some m 2^-53 of itself. F64: the
// mean and the squares about it of the elements less the first one, joined pairwise.
template <class T>
struct Moments {
    double n, a, b;
    __device__ __forceinline__ void add(const Moments &o) {
        if constexpr (!std::is_same_v<T, double>) {
            n += o.n, a += o.a, b += o.b;
        } else if (o.n > 0) {
            const double all = n + o.n, d = o.a - a;
            a += d * (o.n / all);
            b += o.b + d * d * (n * (o.n / all));
            n = all;
        }
    }
    __device__ __forceinline__ double mean(double less) const { return less + (std::is_same_v<T, double> ? a : a / n); }
    __device__ __forceinline__ double variance() const {
        if constexpr (std::is_same_v<T, double>) return b / n;
        const double squares = n * b, square = a * a;
        const double v = ((squares - square) + (__builtin_fma(n, b, -squares) - __builtin_fma(a, a, -square))) / (n * n);
        return v < 0 ? 0 : v;
    }
};

// What a group's elements are taken less: 16-bit ones nothing, others the first one, unless that is infinite or NaN (the
// mean then is).
template <class T>
__device__ __forceinline__ double less_of(const NormArgs &a, int64_t n, int64_t g) {
    if constexpr (sizeof(T) == 2) return 0;
    else {
        const double first = static_cast<double>(reinterpret_cast<const T *>(a.src.p)[n * a.src.sn + g * a.W]);
        return first - first == 0 ? first : 0;
    }
}

struct MapsArgs {
    NormArgs a;
    MapsPlan p;
    int32_t activation;
    void *room;
};

// The workgroup's place: which map, which chunk of its positions, which block of channels; and the lane's.
template <int V>
struct Place {
    int64_t n, chunk, block, s0;  // s0: its first position
    int64_t c0, c1;                   // channels of the block
    int slot;
    int64_t c;  // the lane's first channel
    bool on;
    __device__ __forceinline__ Place(const NormArgs &a, const MapsPlan &p) {
        block = blockIdx.x % p.blocks;
        chunk = blockIdx.x / p.blocks % p.chunks, n = blockIdx.x / p.blocks / p.chunks;
        s0 = chunk * p.run;
        c0 = block * p.lanes * V, c1 = c0 + p.lanes * V < a.C ? c0 + p.lanes * V : a.C;
        slot = threadIdx.x / p.lanes;
        c = c0 + threadIdx.x % p.lanes * V;
        on = slot < p.slots && c < a.C;
    }
};

constexpr int kAtOnce = 2;  // positions of a lane requested at a time (with 4 [16, 4096, 320] bf16 takes 32.4 us for 30.5, backwards 2 % more)

// A lane's walk through its positions of one or two maps: the next vectors are under way while f works on these, the first
// ones from the walk's beginning on.
template <class T, int V, int MAPS>
struct Walk {
    const T *from[MAPS];
    int64_t step[MAPS], s, S, round;  // between positions; the next run's first position of the lane, the map's, from run to run
    int slots;
    Vec<T, V> next[MAPS][kAtOnce];

    __device__ __forceinline__ Walk(const Place<V> &at, const NormArgs &a, const MapsPlan &p, const Maps &x, const Maps &y)
        : s(at.s0 + at.slot), S(at.on ? a.S : 0), round(p.run * p.chunks), slots(p.slots) {
        from[0] = reinterpret_cast<const T *>(x.p) + at.n * x.sn + at.c, step[0] = x.ss;
        if constexpr (MAPS == 2) from[1] = reinterpret_cast<const T *>(y.p) + at.n * y.sn + at.c, step[1] = y.ss;
        fetch();
    }
    __device__ __forceinline__ void fetch() {
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
            if (s + k * slots < S) {
#pragma unroll
                for (int j = 0; j < MAPS; ++j) next[j][k].load(from[j] + (s + k * slots) * step[j]);
            }
        }
    }
    // Calls f for every position, and done() after every kAtOnce of them.
    template <class F, class D>
    __device__ __forceinline__ void run(F f, D done) {
        while (s < S) {
            Vec<T, V> now[MAPS][kAtOnce];
#pragma unroll
            for (int j = 0; j < MAPS; ++j) {
#pragma unroll
                for (int k = 0; k < kAtOnce; ++k) now[j][k] = next[j][k];
            }
            const int64_t here = s;
            s += round;
            fetch();
#pragma unroll
            for (int k = 0; k < kAtOnce; ++k) {
                if (here + k * slots < S) {
                    if constexpr (MAPS == 2) f(here + k * slots, now[0][k], now[1][k]);
                    else f(here + k * slots, now[0][k]);
                }
            }
            done();
        }
    }
    template <class F>
    __device__ __forceinline__ void run(F f) {
        run(f, [] {});
    }
};

// ---- forwards ---------------------------------------------------------------------------------------------------------

// [N][chunks][G + blocks] moments; block b writes those of the groups g that it has channels of, at b + g (of two blocks
// one group at most is both's).
template <class T, int V>
__global__ void __launch_bounds__(kBlock) moments_kernel(MapsArgs m) {
    const NormArgs &a = m.a;
    const Place<V> at(a, m.p);
    Walk<T, V, 1> walk(at, a, m.p, a.src, a.src);
    // Of each of the lane's channels. F64 sums about the first one that the lane meets.
    double n = 0, sum[V], squares[V], about[V], less[V];
    int64_t g = at.c / a.W, in = at.c - g * a.W;  // the channel's group, and its place there
#pragma unroll
    for (int i = 0; i < V; ++i) {
        sum[i] = squares[i] = about[i] = 0;
        less[i] = at.on ? less_of<T>(a, at.n, g) : 0;
        if (++in == a.W) in = 0, ++g;
    }
    walk.run([&](int64_t, const Vec<T, V> &x) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            double v = x.get(i);
            if constexpr (sizeof(T) > 2) v -= less[i];
            if constexpr (std::is_same_v<T, double>) {
                if (n == 0) about[i] = v;
                v -= about[i];
            }
            sum[i] += v, squares[i] = __builtin_fma(v, v, squares[i]);
        }
        n += 1;
    });
    __shared__ double slots_sum[kBlock][V], slots_squares[kBlock][V], slots_n[kBlock];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        if constexpr (std::is_same_v<T, double>) {
            const double shift = n > 0 ? sum[i] / n : 0;
            slots_sum[threadIdx.x][i] = about[i] + shift;
            slots_squares[threadIdx.x][i] = squares[i] - shift * sum[i];
        } else {
            slots_sum[threadIdx.x][i] = sum[i], slots_squares[threadIdx.x][i] = squares[i];
        }
    }
    slots_n[threadIdx.x] = n;
    __syncthreads();
    // The slots of a channel joined by `share` threads, then those; the result goes to the first slot's place.
    __shared__ Moments<T> parts[kBlock];
    const int channels = static_cast<int>(at.c1 - at.c0), share = channels < kBlock ? kBlock / channels : 1;
    for (int k = threadIdx.x; k < channels * share; k += kBlock) {
        const int c = k % channels;
        Moments<T> all{0, 0, 0};
        for (int slot = k / channels; slot < m.p.slots; slot += share) {
            const int l = c / V + slot * m.p.lanes;
            all.add(Moments<T>{slots_n[l], slots_sum[l][c % V], slots_squares[l][c % V]});
        }
        if (share == 1) slots_sum[c / V][c % V] = all.a, slots_squares[c / V][c % V] = all.b;
        else parts[k] = all;
    }
    __syncthreads();
    if (share > 1) {
        if (threadIdx.x < static_cast<unsigned>(channels)) {
            const int c = threadIdx.x;
            Moments<T> all = parts[c];
            for (int k = 1; k < share; ++k) all.add(parts[c + k * channels]);
            slots_sum[c / V][c % V] = all.a, slots_squares[c / V][c % V] = all.b;
        }
        __syncthreads();
    }
    // The positions of the workgroup's runs.
    const int64_t rounds = a.S / (m.p.run * m.p.chunks), left = a.S - rounds * m.p.run * m.p.chunks - at.s0;
    const double positions = static_cast<double>(rounds * m.p.run + (left < 0 ? 0 : (left < m.p.run ? left : m.p.run)));
    Moments<T> *out = static_cast<Moments<T> *>(m.room) + (at.n * m.p.chunks + at.chunk) * (a.G + m.p.blocks) + at.block;
    for (int64_t g = at.c0 / a.W + threadIdx.x; g * a.W < at.c1; g += kBlock) {
        const int64_t from = g * a.W > at.c0 ? g * a.W : at.c0, to = (g + 1) * a.W < at.c1 ? (g + 1) * a.W : at.c1;
        Moments<T> all{0, 0, 0};
        for (int64_t c = from - at.c0; c < to - at.c0; ++c) all.add(Moments<T>{positions, slots_sum[c / V][c % V], slots_squares[c / V][c % V]});
        out[g] = all;
    }
}

// The groups' means and reciprocal deviations, [N * G][2] of f64 behind the moments, a wave a group: in the second pass's
// workgroups the same sums took longer than this launch does ([16, 4096, 320] bf16: 21 us with them).
template <class T>
__global__ void __launch_bounds__(kBlock) statistics_kernel(MapsArgs m, double *statistics) {
    using C = typename Comp<T>::C;
    const NormArgs &a = m.a;
    const int64_t group = static_cast<int64_t>(blockIdx.x) * (kBlock / 64) + threadIdx.x / 64;
    if (group >= a.N * a.G) return;
    const int64_t n = group / a.G, g = group - n * a.G, block_channels = static_cast<int64_t>(m.p.lanes) * m.p.v;
    const int lane = threadIdx.x % 64;
    const Moments<T> *in = static_cast<const Moments<T> *>(m.room) + n * m.p.chunks * (a.G + m.p.blocks) + g;
    Moments<T> all{0, 0, 0};
    for (int64_t b = g * a.W / block_channels; b <= ((g + 1) * a.W - 1) / block_channels; ++b) {
        constexpr int kAhead = 4;  // loads in flight
        for (int64_t k = lane; k < m.p.chunks; k += kAhead * 64) {
            Moments<T> some[kAhead];
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                if (k + j * 64 < m.p.chunks) some[j] = in[(k + j * 64) * (a.G + m.p.blocks) + b];
            }
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                if (k + j * 64 < m.p.chunks) all.add(some[j]);
            }
        }
    }
    for (int d = 1; d < 64; d <<= 1) {
        const Moments<T> other{__shfl_xor(all.n, d, 64), __shfl_xor(all.a, d, 64), __shfl_xor(all.b, d, 64)};
        // Joined lower lane first on both sides, so that they agree.
        Moments<T> low = lane & d ? other : all;
        low.add(lane & d ? all : other);
        all = low;
    }
    if (lane != 0) return;
    const double mean = all.mean(less_of<T>(a, n, g)), rstd = reciprocal_root(all.variance() + a.eps);
    statistics[2 * group] = mean, statistics[2 * group + 1] = rstd;
    if (a.mean.p != nullptr) reinterpret_cast<C *>(a.mean.p)[a.mean.at(n, g)] = static_cast<C>(mean);
    if (a.rstd.p != nullptr) reinterpret_cast<C *>(a.rstd.p)[a.rstd.at(n, g)] = static_cast<C>(rstd);
}

template <class T, int V, bool PAST>
__global__ void __launch_bounds__(kBlock) apply_kernel(MapsArgs m, const double *statistics) {
    using C = typename Comp<T>::C;
    const NormArgs &a = m.a;
    const Place<V> at(a, m.p);
    if (!at.on) return;
    Walk<T, V, 1> walk(at, a, m.p, a.src, a.src);
    // (x - near) * w + b, the weight with the reciprocal deviation and the bias with what the subtraction leaves of the mean.
    C w[V], b[V], near[V];
    load_channels<T, V>(a.weight, at.c, C(1), w);
    load_channels<T, V>(a.bias, at.c, C(0), b);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const double *p = statistics + 2 * (at.n * a.G + (at.c + i) / a.W);
        near[i] = static_cast<C>(p[0]);
        b[i] = static_cast<C>(__builtin_fma((static_cast<double>(near[i]) - p[0]) * p[1], static_cast<double>(w[i]), static_cast<double>(b[i])));
        w[i] = static_cast<C>(p[1] * static_cast<double>(w[i]));
    }
    T *to = reinterpret_cast<T *>(a.out.p) + at.n * a.out.sn + at.c;
    walk.run([&](int64_t s, const Vec<T, V> &x) {
        C z[V];
#pragma unroll
        for (int i = 0; i < V; ++i) z[i] = fma_(x.get(i) - near[i], w[i], b[i]);
        activate_all<T, V>(m.activation, z);
        Vec<T, V> y;
        y.round(z);
        y.template store<PAST>(to + s * a.out.ss);
    });
}

// ---- backwards --------------------------------------------------------------------------------------------------------

// hat, and in z the derivative of what it leads to.
template <class T, int V, class C>
__device__ __forceinline__ void hat_and_slope(int32_t activation, const Vec<T, V> &x, const C (&mean)[V], const C (&rstd)[V], const C (&w)[V],
                                              const C (&b)[V], C (&hat)[V], C (&z)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
        hat[i] = (x.get(i) - mean[i]) * rstd[i];
        z[i] = fma_(hat[i], w[i], b[i]);
    }
    slope_all<T, V>(activation, z);
}
template <class T, int V, class C>
__device__ __forceinline__ void load_statistics(const NormArgs &a, int64_t n, int64_t c, C (&mean)[V], C (&rstd)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int64_t g = (c + i) / a.W;
        mean[i] = reinterpret_cast<const C *>(a.mean.p)[a.mean.at(n, g)], rstd[i] = reinterpret_cast<const C *>(a.rstd.p)[a.rstd.at(n, g)];
    }
}

// Rows of sums per channel, [2][N * chunks][C]: of d * hat, and of d.
template <class T, int V>
__global__ void __launch_bounds__(kBlock) channel_sums_kernel(MapsArgs m) {
    using C = typename Comp<T>::C;
    const NormArgs &a = m.a;
    const Place<V> at(a, m.p);
    Walk<T, V, 2> walk(at, a, m.p, a.src, a.grad);
    constexpr bool kRuns = sizeof(C) == 4;
    static_assert(kMostRun % kAtOnce == 0, "a run ends where the walk's steps end");
    C sum[V], sum_h[V], all[kRuns ? V : 1], all_h[kRuns ? V : 1];
    int run = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        sum[i] = sum_h[i] = 0;
        if constexpr (kRuns) all[i] = all_h[i] = 0;
    }
    if (at.on) {
        C w[V], b[V], mean[V], rstd[V];
        load_channels<T, V>(a.weight, at.c, C(1), w);
        load_channels<T, V>(a.bias, at.c, C(0), b);
        load_statistics<T, V>(a, at.n, at.c, mean, rstd);
        walk.run([&](int64_t, const Vec<T, V> &x, const Vec<T, V> &dy) {
            C hat[V], z[V];
            hat_and_slope<T, V>(m.activation, x, mean, rstd, w, b, hat, z);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const C d = dy.get(i) * z[i];
                sum[i] += d, sum_h[i] = fma_(d, hat[i], sum_h[i]);
            }
        }, [&] {
            if constexpr (kRuns) {
                run += kAtOnce;
                if (run == kMostRun) {
                    run = 0;
#pragma unroll
                    for (int i = 0; i < V; ++i) add_run(all[i], sum[i]), add_run(all_h[i], sum_h[i]);
                }
            }
        });
    }
    __shared__ C slots[2][kBlock][V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        if constexpr (kRuns) sum[i] += all[i], sum_h[i] += all_h[i];
        slots[0][threadIdx.x][i] = sum_h[i], slots[1][threadIdx.x][i] = sum[i];
    }
    __syncthreads();
    C *out = static_cast<C *>(m.room);
    const int64_t rows = a.N * m.p.chunks, part = at.n * m.p.chunks + at.chunk;
    __shared__ double parts[kBlock];
    const int channels = static_cast<int>(at.c1 - at.c0), share = channels < kBlock ? kBlock / channels : 1;
    for (int which = 0; which < 2; ++which) {
        for (int k = threadIdx.x; k < channels * share; k += kBlock) {
            const int c = k % channels;
            double total = 0;
            for (int slot = k / channels; slot < m.p.slots; slot += share) total += slots[which][c / V + slot * m.p.lanes][c % V];
            if (share == 1) out[(which * rows + part) * a.C + at.c0 + c] = static_cast<C>(total);
            else parts[k] = total;
        }
        if (share > 1) {
            __syncthreads();
            if (threadIdx.x < static_cast<unsigned>(channels)) {
                double total = 0;
                for (int k = 0; k < share; ++k) total += parts[threadIdx.x + k * channels];
                out[(which * rows + part) * a.C + at.c0 + threadIdx.x] = static_cast<C>(total);
            }
            __syncthreads();
        }
    }
}

// The means over each group, [N * G][2] of f64 behind the rows: of weight * d, and of weight * d * hat, a workgroup a group;
// and, by the workgroups after those, the weights' gradients.
template <class T>
__global__ void __launch_bounds__(kBlock) join_kernel(MapsArgs m, double *means) {
    using C = typename Comp<T>::C;
    const NormArgs &a = m.a;
    if (blockIdx.x >= a.N * a.G) return sum_channels<T>(a, static_cast<const C *>(m.room), a.N * m.p.chunks, blockIdx.x - a.N * a.G);
    const int64_t n = blockIdx.x / a.G, g = blockIdx.x % a.G, parts = a.N * m.p.chunks;
    const C *in = static_cast<const C *>(m.room);
    double sum = 0, sum_h = 0;
    // Lanes across the group's channels, the rest of the workgroup along its chunks, eight loads of each kind in flight.
    const int across = a.W < kBlock ? static_cast<int>(a.W) : kBlock, slots = kBlock / across, slot = threadIdx.x / across;
    for (int64_t in_group = threadIdx.x % across; in_group < a.W && slot < slots; in_group += across) {
        const int64_t c = g * a.W + in_group;
        const double w = weight_of<T>(a.weight, c);
        const C *rows = in + n * m.p.chunks * a.C + c;
        constexpr int kAhead = 8;
        for (int64_t k = slot; k < m.p.chunks; k += kAhead * slots) {
            C d[kAhead], dh[kAhead];
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                const int64_t part = k + j * slots;
                d[j] = dh[j] = 0;
                if (part < m.p.chunks) dh[j] = rows[part * a.C], d[j] = rows[(parts + part) * a.C];
            }
#pragma unroll
            for (int j = 0; j < kAhead; ++j) sum += w * d[j], sum_h += w * dh[j];
        }
    }
    sum = lanes_sum(sum, 64), sum_h = lanes_sum(sum_h, 64);
    __shared__ double waves[2][kBlock / 64];
    if (threadIdx.x % 64 == 0) waves[0][threadIdx.x / 64] = sum, waves[1][threadIdx.x / 64] = sum_h;
    __syncthreads();
    if (threadIdx.x < 2) {
        double total = 0;
#pragma unroll
        for (int k = 0; k < kBlock / 64; ++k) total += waves[threadIdx.x][k];
        means[2 * blockIdx.x + threadIdx.x] = total / (static_cast<double>(a.S) * static_cast<double>(a.W));
    }
}

template <class T, int V, bool PAST>
__global__ void __launch_bounds__(kBlock) apply_back_kernel(MapsArgs m, const double *means) {
    using C = typename Comp<T>::C;
    const NormArgs &a = m.a;
    const Place<V> at(a, m.p);
    if (!at.on) return;
    Walk<T, V, 2> walk(at, a, m.p, a.src, a.grad);
    C w[V], b[V], mean[V], rstd[V], d_mean[V], dh_mean[V];
    load_channels<T, V>(a.weight, at.c, C(1), w);
    load_channels<T, V>(a.bias, at.c, C(0), b);
    load_statistics<T, V>(a, at.n, at.c, mean, rstd);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const double *p = means + 2 * (at.n * a.G + (at.c + i) / a.W);
        d_mean[i] = static_cast<C>(p[0]), dh_mean[i] = static_cast<C>(p[1]);
    }
    T *to = reinterpret_cast<T *>(a.out.p) + at.n * a.out.sn + at.c;
    walk.run([&](int64_t s, const Vec<T, V> &x, const Vec<T, V> &dy) {
        C hat[V], z[V];
        hat_and_slope<T, V>(m.activation, x, mean, rstd, w, b, hat, z);
#pragma unroll
        for (int i = 0; i < V; ++i) z[i] = rstd[i] * fma_(-hat[i], dh_mean[i], w[i] * (dy.get(i) * z[i]) - d_mean[i]);
        Vec<T, V> dx;
        dx.round(z);
        dx.template store<PAST>(to + s * a.out.ss);
    });
}

int64_t up16(int64_t bytes) { return (bytes + 15) / 16 * 16; }
int64_t rows_bytes(const NormArgs &a, const MapsPlan &p, int32_t dtype) {
    return up16(2 * a.N * p.chunks * a.C * dtype_size(wide_type(dtype)));
}

int64_t moments_bytes(const NormArgs &a, const MapsPlan &p) {
    return up16(a.N * p.chunks * (a.G + p.blocks) * static_cast<int64_t>(3 * sizeof(double)));
}

template <class T, int V>
void launch_maps(hipStream_t stream, const MapsArgs &m, bool backward, bool past) {
    const NormArgs &a = m.a;
    const uint32_t groups = static_cast<uint32_t>(a.N * m.p.chunks * m.p.blocks);
    if (!backward) {
        moments_kernel<T, V><<<groups, kBlock, 0, stream>>>(m);
        double *statistics = reinterpret_cast<double *>(static_cast<char *>(m.room) + moments_bytes(a, m.p));
        statistics_kernel<T><<<static_cast<uint32_t>((a.N * a.G + kBlock / 64 - 1) / (kBlock / 64)), kBlock, 0, stream>>>(m, statistics);
        if (past) apply_kernel<T, V, true><<<groups, kBlock, 0, stream>>>(m, statistics);
        else apply_kernel<T, V, false><<<groups, kBlock, 0, stream>>>(m, statistics);
        return;
    }
    double *means = reinterpret_cast<double *>(static_cast<char *>(m.room) + rows_bytes(a, m.p, sizeof(T) == 2 ? HMR_BF16 : (sizeof(T) == 4 ? HMR_F32 : HMR_F64)));
    channel_sums_kernel<T, V><<<groups, kBlock, 0, stream>>>(m);
    const int64_t summing = a.d_weight.p != nullptr || a.d_bias.p != nullptr ? (a.C + kSumChannels - 1) / kSumChannels : 0;
    join_kernel<T><<<static_cast<uint32_t>(a.N * a.G + summing), kBlock, 0, stream>>>(m, means);
    if (past) apply_back_kernel<T, V, true><<<groups, kBlock, 0, stream>>>(m, means);
    else apply_back_kernel<T, V, false><<<groups, kBlock, 0, stream>>>(m, means);
}

}  // namespace

MapsPlan maps_plan(const NormArgs &a, int32_t dtype) {
    MapsPlan p{};
    const int full = 16 / dtype_size(dtype);
    p.v = a.C % full == 0 ? full : (full == 8 && a.C % 2 == 0 ? 2 : 1);
    const int64_t across = a.C / p.v;
    p.lanes = static_cast<int32_t>(across < kBlock ? across : kBlock);
    p.slots = kBlock / p.lanes;
    p.blocks = (across + p.lanes - 1) / p.lanes;
    // Two workgroups for every compute unit, all of them resident: each one's prologue and sums cost the same however few
    // positions it has ([16, 4096, 320] bf16: 30.5 us, with four 31.7; the gradient of [4, 9216, 512] f32 73 and 74).
    p.run = kAtOnce * p.slots;
    const int64_t most = (a.S + p.run - 1) / p.run;
    int64_t chunks = (512 + a.N * p.blocks - 1) / (a.N * p.blocks);
    p.chunks = chunks < 1 ? 1 : (chunks > most ? most : chunks);
    return p;
}

namespace {
// Short maps of huge groups would leave rows of sums as large as themselves; so many workgroups do not make a launch.
bool maps_fit(const NormArgs &a, int32_t dtype) {
    if (a.N == 0 || a.S == 0 || a.C == 0) return false;
    if (a.S < 8 && a.N * a.C > (int64_t{1} << 22)) return false;
    const MapsPlan p = maps_plan(a, dtype);
    return fits_launch(a.N * p.chunks * p.blocks, kBlock) && fits_launch(a.N * a.G + a.C, kBlock);
}
}  // namespace

int64_t norm_maps_room(const NormArgs &a, int32_t dtype, bool backward) {
    if (!maps_fit(a, dtype)) return 0;
    const MapsPlan p = maps_plan(a, dtype);
    return (backward ? rows_bytes(a, p, dtype) : moments_bytes(a, p)) + a.N * a.G * static_cast<int64_t>(2 * sizeof(double));
}

bool queue_norm_maps(hipStream_t stream, int32_t dtype, const NormArgs &a, int32_t activation, void *room, bool backward) {
    if (!channels_adjacent(a, backward) || !maps_fit(a, dtype)) return false;
    MapsArgs m{a, maps_plan(a, dtype), activation, room};
    // The second pass finds the maps in the memory-side cache if its results do not push them out: from half of what that
    // holds on they are stored past it ([4, 9216, 512] f32 backwards, 226 MB: 79 us through the caches, 73 past them).
    const bool past = a.N * a.S * a.C * dtype_size(dtype) * (backward ? 3 : 2) > kCacheResidentBytes / 2;
    with_float_type(dtype, [&](auto tag) {
        using T = typename decltype(tag)::type;
        constexpr int kFull = 16 / static_cast<int>(sizeof(T));
        if (m.p.v == kFull) launch_maps<T, kFull>(stream, m, backward, past);
        else if (kFull == 8 && m.p.v == 2) launch_maps<T, kFull == 8 ? 2 : 1>(stream, m, backward, past);
        else launch_maps<T, 1>(stream, m, backward, past);
    });
    return true;
}

}  // namespace nn
}  // namespace hmr
