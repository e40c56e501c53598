// group_norm.cu -- group norm with an activation, channels last, forward and backward.
//
// x[n][s][c], group g = c / D, D = channels / groups, m = positions * D elements per (n, g):
//   mean = sum x / m, var = sum (x - mean)^2 / m, r = 1 / sqrt(var + eps), h = (x - mean) r,
//   z = h w + b, y = act(z);
// backward: dz = dy act'(z), db = sum dz, dw = sum dz h (over n and s),
//   c1 = sum_g dz w / m, c2 = sum_g dz w h / m, dx = r (dz w - c1 - h c2).
//
// All of it is bound by memory: x (and dy) in, y (dx) out.  Three ways to read the inputs once:
//   * warp form: a group of at most 512 elements sits in the registers of 4 to 32 lanes;
//   * slab form: a block of whole groups of one n sits in the shared memory of a cluster of CTAs;
//   * stream form, for what fits neither: one pass for sums of row chunks, one that applies them.
// Measured (graph replays, inputs beyond L2 or resident as a layer's are):
//   warp form, 8192 x 4096, groups of 128, ReLU, F32: forward 49 us = 5.5 TB/s (0.84 of a copy's 6.55), backward
//     87 us = 4.6 TB/s with the parameters' gradients; 54 and 60 % of the issue slots are taken by 22 warps an SM,
//     which the registers leave: too few to cover each other's latencies; BF16 39 and 84 us;
//   slab form, BF16, SiLU: forward 5 x 4095 x 320 15.7 us, one CTA an SM, a chain of load, sums, cluster, stores;
//     backward 16 x 1024 x 640 36 us, 52 % of the slots by 22 % of the warps: some 50 instructions an element, half of them the
//     SiLU slope, which is formed twice because dz does not fit beside x and dy;
//   stream form: reads twice; 35 us against the slab form's 21 on a map that both take.
// The variance is taken about the mean in every form: the warp form has it before it sums the squares; a thread of
// the slab and stream forms takes its rows' about the mean of those before (row_moments), and threads, channels,
// CTAs and chunks are joined about their joint means.
#include <algorithm>
#include <numeric>

#include "learn.cuh"
#include "provider.h"
#include "tma.cuh"

namespace pcu {

constexpr int kNormThreads = 256;
// Warp form: CTAs per SM that walk over the batch at once, by the bytes of a lane's elements in the wide
// type: forward a lane keeps them and two parameters each, backward also dy and two sums.
__host__ __device__ constexpr int warp_form_ctas(int bytes, bool backward) {
    return backward ? (bytes <= 32 ? 3 : bytes <= 64 ? 2 : 1) : (bytes <= 64 ? 3 : 1);
}

// A channels-last tensor: element (n, s, c) at n * batch + s * row + c.
template <typename T> struct Maps {
    T *base;
    uint64_t batch, row;
    __device__ __forceinline__ T *at(uint64_t n, uint64_t s, uint64_t c) const { return base + n * batch + s * row + c; }
};

// How a call is carried out; a function of the sizes and of whether 16-byte accesses are possible.
struct NormPlan {
    enum Form { kWarp, kSlab, kStream } form;
    int vector;                // elements per access
    int per_lane, lanes;       // warp form: accesses per lane, lanes per group (a power of two)
    unsigned items, slices;    // accesses per group; parts of the batch
    unsigned block_groups, blocks, ranks, threads;  // slab form: groups per cluster, of one n; CTAs
    unsigned slab_rows;
    size_t slab_bytes, shared;  // of one tensor's slab; of the CTA
    unsigned tiles, tile, chunks;  // stream form: column tiles of `tile` accesses, row chunks
    uint64_t chunk_rows;
    uint64_t partial_rows;                 // parameters' gradients: partial sums [rows][2][channels]
    uint64_t workspace;                    // elements of the wide type
};

template <typename T> struct NormParams {
    using W = WideOf<T>;
    Maps<const T> x, dy;
    Maps<T> out;  // y, or dx
    const W *weight, *bias;
    W *stats_out;
    const W *stats;
    W *partial;  // workspace: partial sums
    W *sums;     // workspace: (c1, c2) for each (n, g), stream form
    W *dweight, *dbias;
    uint64_t batch, positions, channels, groups, width;
    W eps;
    int activation;
    NormPlan plan;
    unsigned long long *status;
    ChainGuard guard;
};

// ---- activations, over the V elements of one access (the choice is the same for a whole launch)

// binary32: the hardware's exponential and reciprocal (each within 2 ulp)
__device__ __forceinline__ float logistic(float z) {
    float q;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(q) : "f"(1.0f + fast_exp2(z * -1.4426950408889634f)));
    return q;
}
__device__ __forceinline__ double logistic(double z) { return 1.0 / (1.0 + exp(-z)); }
__device__ __forceinline__ float normal_density(float z) {
    return fast_exp2(z * z * -0.72134752044448170f) * 0.39894228040143267794f;
}
__device__ __forceinline__ double normal_density(double z) { return exp(-0.5 * z * z) * 0.39894228040143267794; }

template <int V, typename W> __device__ __forceinline__ void activate(int act, W (&z)[V]) {
    if (act == PCU_B200_ACTIVATION_RELU) {
#pragma unroll
        for (int e = 0; e < V; ++e) z[e] = z[e] < W(0) ? W(0) : z[e];  // NaN stays
    } else if (act == PCU_B200_ACTIVATION_SILU) {
#pragma unroll
        for (int e = 0; e < V; ++e) z[e] *= logistic(z[e]);
    } else if (act == PCU_B200_ACTIVATION_GELU) {
#pragma unroll
        for (int e = 0; e < V; ++e) z[e] *= W(0.5) * erfc(z[e] * W(-0.70710678118654752440));
    }
}

// h and dz = dy act'(z), z = h w + b.  ReLU's slope is a step.  z is off by at most 2^-21 |h w| and its own
// rounding, so its sign is right where |z| > 2^-19 |b|; the few others are decided in binary64.  A masked
// upstream gradient gives 0, whatever it is.
template <int V, typename W>
__device__ __forceinline__ void bend(int act, const W (&x)[V], const W (&dy)[V], const W (&mean)[V], const W (&r)[V],
                                     const W (&w)[V], const W (&b)[V], W (&h)[V], W (&dz)[V]) {
#pragma unroll
    for (int e = 0; e < V; ++e) h[e] = (x[e] - mean[e]) * r[e], dz[e] = dy[e];
    if (act == PCU_B200_ACTIVATION_RELU) {
        bool near = false;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const W z = fma(h[e], w[e], b[e]);
            if (sizeof(W) == 4) near |= fabs(z) <= fabs(b[e]) * W(0x1p-19);
            dz[e] = z > W(0) ? dy[e] : W(0);
        }
        if (near)
#pragma unroll
            for (int e = 0; e < V; ++e)
                dz[e] = ((double)x[e] - (double)mean[e]) * (double)r[e] * (double)w[e] + (double)b[e] > 0.0 ? dy[e] : W(0);
    } else if (act == PCU_B200_ACTIVATION_SILU) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const W z = h[e] * w[e] + b[e], q = logistic(z);
            dz[e] *= q * (W(1) + z * (W(1) - q));
        }
    } else if (act == PCU_B200_ACTIVATION_GELU) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const W z = h[e] * w[e] + b[e];
            dz[e] *= W(0.5) * erfc(z * W(-0.70710678118654752440)) + z * normal_density(z);
        }
    }
}

// ---- accesses of V elements: 16 bytes, or one element

template <typename T, int V> struct Access {
    using W = WideOf<T>;
    uint4 raw;
    static __device__ __forceinline__ Access load(const T *p) { return {__ldcs(reinterpret_cast<const uint4 *>(p))}; }
    __device__ __forceinline__ void open(W (&v)[V]) const { unpack<T>(raw, v); }
};
template <typename T> struct Access<T, 1> {
    using W = WideOf<T>;
    T raw;
    static __device__ __forceinline__ Access load(const T *p) { return {*p}; }
    __device__ __forceinline__ void open(W (&v)[1]) const { v[0] = Elem<T>::load(raw); }
};

// Stores V elements; what is not finite is recorded, the first of them being event().
template <typename T, int V, typename E>
__device__ __forceinline__ void put(T *to, const WideOf<T> (&v)[V], unsigned long long *status, E event) {
    unsigned bad;
    if constexpr (V == 1) {
        const T y = Elem<T>::round(v[0]);
        *to = y;
        bad = result_kind(Elem<T>::load(y));
    } else {
        const uint4 y = pack<T>(v);
        __stcs(reinterpret_cast<uint4 *>(to), y);
        if constexpr (sizeof(T) >= 4) {  // 0 times an infinity or NaN is NaN, and stays
            WideOf<T> sum = 0;
#pragma unroll
            for (int e = 0; e < V; ++e) sum = fma(v[e], WideOf<T>(0), sum);
            bad = sum != WideOf<T>(0);
        } else {
            bad = not_finite<T>(y);  // rounding can make an infinity
        }
    }
    if (bad) {
        const uint64_t first = event();
        for (int e = 0; e < V; ++e)
            if (const unsigned kind = result_kind(Elem<T>::load(Elem<T>::round(v[e])))) record_fault(status, first + e, kind);
    }
}

template <int V, typename W> __device__ __forceinline__ void parameters(const W *p, uint64_t c, W none, W (&v)[V]) {
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = p ? p[c + e] : none;
}

// 1 / sqrt(var + eps), within 2 ulp in binary32.  A variance that is not finite has no reciprocal root to
// scale by: NaN, not 0.
__device__ __forceinline__ float root(float var, float eps) { return isfinite(var) ? rsqrtf(var + eps) : NAN; }
__device__ __forceinline__ double root(double var, double eps) { return isfinite(var) ? 1.0 / sqrt(var + eps) : NAN; }

// A sum of squares that rounding made negative is 0; NaN stays.
template <typename W> __device__ __forceinline__ W not_negative(W v) { return v < W(0) ? W(0) : v; }

// The mean of each of `rows` rows' V channels, and the sum of squares about it, in one pass; 0 without rows.
// next(x) brings the rows one by one.  A block of rows is summed about the mean of the rows before it (the first
// about the first row): with d = x - mean, a block's sums s of d and q of d^2 and the rows n up to its end, q - s^2 / n
// is what the block adds to the squares, both for it and for the mean's move by s / n.  A far first row so costs the
// first block some digits and no more, where one sum about it over 7,000 rows left the squares 2 % off.
// LONG, for thousands of rows: blocks of 16, each one's squares summed by themselves.  Else, for up to some hundred:
// blocks that end at 32, 256, ... rows, on top of the squares before them (most threads have fewer than 32 rows;
// blocks of 16 cost a forward pass of 16 x 4095 x 1280 BF16 1.5 %).
template <int V, bool LONG, typename W, typename Next>
__device__ __forceinline__ void row_moments(int rows, Next next, W (&mean)[V], W (&square)[V]) {
#pragma unroll
    for (int e = 0; e < V; ++e) mean[e] = square[e] = W(0);
    if (rows > 0) next(mean);
    for (int done = 1; done < rows;) {
        const int end = min(rows, LONG ? (done / 16 + 1) * 16 : done < 32 ? 32 : 8 * done);
        W sum[V] = {}, block[V] = {}, x[V];
        W(&squares)[V] = LONG ? block : square;
        // 16 elements on their way: more rows of 8 cost registers that other warps need (8 x 32768 x 320 BF16 188 us
        // with two rows, 200 with four), single elements want more (300 x 2048 x 256 F32 in rows of 257 1367 us with
        // 16 rows, 1567 with four)
#pragma unroll 16 / V
        for (; done < end; ++done) {
            next(x);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const W d = x[e] - mean[e];
                sum[e] += d;
                squares[e] += d * d;
            }
        }
        const W inverse = W(1) / (W)done;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const W shift = sum[e] * inverse;
            const W about = not_negative(squares[e] - sum[e] * shift);
            square[e] = LONG ? square[e] + about : about;
            mean[e] += shift;
        }
    }
}

// ---- warp form
//
// `lanes` lanes hold a group, K accesses each; 32 / lanes adjacent groups per warp.  A warp keeps its
// groups and walks over the batch, U at a time for loads in flight, so that the parameters stay in
// registers, and their gradients too: each warp ends with one partial sum per element of its groups.
template <typename T, int V, int K> struct WarpGroup {
    using W = WideOf<T>;
    int sub;
    uint64_t slice, g;
    bool active, there[K];
    W w[K][V], b[K][V];

    __device__ __forceinline__ bool place(const NormParams<T> &p) {
        const NormPlan &plan = p.plan;
        const int lane = threadIdx.x % 32, per = 32 / plan.lanes;
        const uint64_t warp = (uint64_t)blockIdx.x * (kNormThreads / 32) + threadIdx.x / 32;
        const uint64_t sets = (p.groups + per - 1) / per;
        if (warp >= sets * plan.slices) return false;
        sub = lane % plan.lanes;
        slice = warp / sets;
        g = warp % sets * per + lane / plan.lanes;
        active = g < p.groups;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            there[k] = active && sub + k * plan.lanes < (int)plan.items;
            unsigned row, channel;
            item(p, k, row, channel);
            parameters<V>(p.weight, channel, W(1), w[k]);
            parameters<V>(p.bias, channel, W(0), b[k]);
        }
        return true;
    }
    // access k's place in a sample; (0, 0) where there is none
    __device__ __forceinline__ void item(const NormParams<T> &p, int k, unsigned &row, unsigned &channel) const {
        const unsigned item = sub + k * p.plan.lanes, across = (unsigned)(p.width / V);
        row = there[k] ? item / across : 0;
        channel = there[k] ? (unsigned)(g * p.width) + item % across * V : 0;
    }
    // its offset from the sample's first element (the plan sees to it that samples span less than 2^31)
    template <typename M> __device__ __forceinline__ int offset(const NormParams<T> &p, const M &maps, int k) const {
        unsigned row, channel;
        item(p, k, row, channel);
        return (int)(row * (unsigned)maps.row + channel);
    }
    __device__ __forceinline__ uint64_t event(const NormParams<T> &p, int k, uint64_t n) const {
        unsigned row, channel;
        item(p, k, row, channel);
        return (n * p.positions + row) * p.channels + channel;
    }
};

template <int U, typename W> __device__ __forceinline__ void lanes_sum(W (&v)[U], int lanes) {
    for (int o = lanes / 2; o; o >>= 1)
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] += __shfl_xor_sync(~0u, v[u], o);
}

template <typename T, int V, int K, int U>
__global__ void __launch_bounds__(kNormThreads, K > 4 ? 1 : warp_form_ctas(V * K * sizeof(WideOf<T>), false)) norm_warp_kernel(const NormParams<T> p) {
    using W = WideOf<T>;
    in_stream_order();
    if (!chain_admits(p.guard)) return;
    WarpGroup<T, V, K> at;
    if (!at.place(p)) return;
    const W inverse = W(1) / (W)(p.positions * p.width);
    const uint64_t stride = (uint64_t)p.plan.slices * U;
    const T *from = p.x.base + at.slice * U * p.x.batch;
    T *to = p.out.base + at.slice * U * p.out.batch;
    int in[K], out[K];
#pragma unroll
    for (int k = 0; k < K; ++k) in[k] = at.offset(p, p.x, k), out[k] = at.offset(p, p.out, k);
    W *stats = p.stats_out + 2 * (at.slice * U * p.groups + at.g);
    for (uint64_t n = at.slice * U; n < p.batch; n += stride) {
        const int here = (int)min((uint64_t)U, p.batch - n);
        W x[U][K][V], mean[U] = {}, square[U] = {};
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if (at.there[k] && u < here) Access<T, V>::load(from + u * p.x.batch + in[k]).open(x[u][k]);
                else
#pragma unroll
                    for (int e = 0; e < V; ++e) x[u][k][e] = W(0);
            }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int e = 0; e < V; ++e) mean[u] += x[u][k][e];
        lanes_sum(mean, p.plan.lanes);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            mean[u] *= inverse;
#pragma unroll
            for (int k = 0; k < K; ++k)
                if (at.there[k])
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        x[u][k][e] -= mean[u];
                        square[u] += x[u][k][e] * x[u][k][e];
                    }
        }
        lanes_sum(square, p.plan.lanes);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (u >= here) break;
            const W r = root(square[u] * inverse, p.eps);
            if (at.sub == 0 && at.active) stats[2 * u * p.groups] = mean[u], stats[2 * u * p.groups + 1] = r;
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if (!at.there[k]) continue;
#pragma unroll
                for (int e = 0; e < V; ++e) x[u][k][e] = x[u][k][e] * r * at.w[k][e] + at.b[k][e];
                activate<V>(p.activation, x[u][k]);
                put<T, V>(to + u * p.out.batch + out[k], x[u][k], p.status, [&] { return at.event(p, k, n + u); });
            }
        }
        from += stride * p.x.batch, to += stride * p.out.batch;
        stats += 2 * stride * p.groups;
    }
}

template <typename T, int V, int K, int U>
__global__ void __launch_bounds__(kNormThreads, K > 4 ? 1 : warp_form_ctas(V * K * sizeof(WideOf<T>), true)) norm_warp_backward_kernel(const NormParams<T> p) {
    using W = WideOf<T>;
    in_stream_order();
    if (!chain_admits(p.guard)) return;
    WarpGroup<T, V, K> at;
    if (!at.place(p)) return;
    const W inverse = W(1) / (W)(p.positions * p.width);
    const uint64_t stride = (uint64_t)p.plan.slices * U;
    const T *from = p.x.base + at.slice * U * p.x.batch, *up = p.dy.base + at.slice * U * p.dy.batch;
    T *to = p.out.base + at.slice * U * p.out.batch;
    int in[K], grad[K], out[K];
#pragma unroll
    for (int k = 0; k < K; ++k) in[k] = at.offset(p, p.x, k), grad[k] = at.offset(p, p.dy, k), out[k] = at.offset(p, p.out, k);
    const W *stats = p.stats + 2 * (at.slice * U * p.groups + (at.active ? at.g : 0));
    W dw[K][V] = {}, db[K][V] = {};
    for (uint64_t n = at.slice * U; n < p.batch; n += stride) {
        const int here = (int)min((uint64_t)U, p.batch - n);
        W x[U][K][V], dy[U][K][V], c1[U] = {}, c2[U] = {}, mean[U], r[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if (at.there[k] && u < here) {
                    Access<T, V>::load(from + u * p.x.batch + in[k]).open(x[u][k]);
                    Access<T, V>::load(up + u * p.dy.batch + grad[k]).open(dy[u][k]);
                } else {
#pragma unroll
                    for (int e = 0; e < V; ++e) x[u][k][e] = dy[u][k][e] = W(0);
                }
            }
            mean[u] = u < here ? stats[2 * u * p.groups] : W(0);
            r[u] = u < here ? stats[2 * u * p.groups + 1] : W(0);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            W means[V], rs[V];
#pragma unroll
            for (int e = 0; e < V; ++e) means[e] = mean[u], rs[e] = r[u];
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if (!at.there[k] || u >= here) continue;
                W h[V], dz[V];
                bend<V>(p.activation, x[u][k], dy[u][k], means, rs, at.w[k], at.b[k], h, dz);
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    dw[k][e] += dz[e] * h[e];
                    db[k][e] += dz[e];
                    const W d = dz[e] * at.w[k][e];
                    c1[u] += d;
                    c2[u] += d * h[e];
                    x[u][k][e] = h[e], dy[u][k][e] = d;
                }
            }
        }
        lanes_sum(c1, p.plan.lanes);
        lanes_sum(c2, p.plan.lanes);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (u >= here) break;
            c1[u] *= inverse, c2[u] *= inverse;
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if (!at.there[k]) continue;
#pragma unroll
                for (int e = 0; e < V; ++e) x[u][k][e] = r[u] * (dy[u][k][e] - c1[u] - x[u][k][e] * c2[u]);
                put<T, V>(to + u * p.out.batch + out[k], x[u][k], p.status, [&] { return at.event(p, k, n + u); });
            }
        }
        from += stride * p.x.batch, up += stride * p.dy.batch, to += stride * p.out.batch;
        stats += 2 * stride * p.groups;
    }
    if (!p.partial) return;
    W *sums = p.partial + 2 * at.slice * p.channels;
    if (p.positions == 1) {
#pragma unroll
        for (int k = 0; k < K; ++k)
            if (at.there[k]) {
                W *mine = sums + at.g * p.width + (at.sub + k * p.plan.lanes) * V;
#pragma unroll
                for (int e = 0; e < V; ++e) mine[e] = dw[k][e], mine[p.channels + e] = db[k][e];
            }
        return;
    }
    // The positions of each channel are summed here, through shared memory: the workspace, and the kernel that
    // adds the slices, would have as many times the rows (138 x 61 x 82, 41 groups, F32: 96 us for 21).
    __shared__ W elements[kNormThreads / 32][32 * K * V];
    W *mine = elements[threadIdx.x / 32];
    const int lane = threadIdx.x % 32, width = (int)p.width, group = (int)p.plan.items * V;
    const uint64_t g0 = at.g - lane / p.plan.lanes;
    const int channels = (int)min((uint64_t)(32 / p.plan.lanes), p.groups - g0) * width;
    auto give = [&](const W (&v)[K][V], W *to) {
        __syncwarp();
#pragma unroll
        for (int k = 0; k < K; ++k)
            if (at.there[k])
#pragma unroll
                for (int e = 0; e < V; ++e) mine[lane / p.plan.lanes * group + (at.sub + k * p.plan.lanes) * V + e] = v[k][e];
        __syncwarp();
        for (int i = lane; i < channels; i += 32) {
            const int g = i / width;
            W all = 0;
            for (int at_ = g * group + i % width; at_ < (g + 1) * group; at_ += width) all += mine[at_];
            to[g0 * width + i] = all;
        }
    };
    give(dw, sums), give(db, sums + p.channels);
}

// ---- columns: the thread mapping of the slab and stream forms
//
// A thread keeps one access of columns and takes every `deep`-th row, so a channel's parameters,
// statistics and sums stay in its registers.

// ---- slab form
//
// A cluster's CTAs hold `slab_rows` rows each of a block of whole groups of one n in shared memory.  A
// thread copies in and reads back only its own accesses.  Sums are joined through the cluster in
// rank order.
template <typename T, int V, int TENSORS> struct Slab {
    using W = WideOf<T>;
    uint64_t n, c0, s0;
    int groups, width, across, deep, tx, ty, rows;
    uint32_t rank, ranks;
    bool active;
    T *mine[TENSORS];  // this thread's first access of each tensor; its next ones are `deep` rows on
    W *scratch, *total, *joined;

    __device__ __forceinline__ void place(const NormParams<T> &p, unsigned char *smem) {
        const NormPlan &plan = p.plan;
        asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
        rank = cluster_rank();
        const unsigned cluster = blockIdx.x / ranks, block = cluster % plan.blocks;
        n = cluster / plan.blocks;
        const uint64_t g0 = (uint64_t)block * plan.block_groups;
        width = (int)p.width;
        groups = (int)min((uint64_t)plan.block_groups, p.groups - g0);
        c0 = g0 * p.width;
        across = groups * width / V;
        deep = (int)blockDim.x / across;
        tx = (int)threadIdx.x % across;
        ty = (int)threadIdx.x / across;
        active = ty < deep;
        s0 = (uint64_t)rank * plan.slab_rows;
        rows = s0 < p.positions ? (int)min((uint64_t)plan.slab_rows, p.positions - s0) : 0;
#pragma unroll
        for (int t = 0; t < TENSORS; ++t)
            mine[t] = reinterpret_cast<T *>(smem + t * plan.slab_bytes) + (ty * across + tx) * V;
        scratch = reinterpret_cast<W *>(smem + TENSORS * plan.slab_bytes);
        total = scratch + 2 * blockDim.x * (V + 1);
        joined = total + 2 * plan.block_groups;
    }
    __device__ __forceinline__ uint64_t channel() const { return c0 + (uint64_t)tx * V; }
    __device__ __forceinline__ int step() const { return deep * across * V; }  // from one access to the next
    __device__ __forceinline__ void bring(int tensor, const Maps<const T> &from) const {
        if (!active) return;
        const T *src = from.at(n, s0 + ty, channel());
        T *dst = mine[tensor];
        const uint64_t stride = deep * from.row;
        for (int r = ty; r < rows; r += deep, src += stride, dst += step()) {
            if (V > 1)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_addr(dst)), "l"(src) : "memory");
            else
                *dst = *src;
        }
    }
    __device__ __forceinline__ static void read(const T *at, W (&v)[V]) {
        if constexpr (V > 1) unpack<T>(*reinterpret_cast<const uint4 *>(at), v);
        else v[0] = Elem<T>::load(*at);
    }
    // One value per channel of each thread's access, for Q quantities, summed over the rows' threads and
    // given to each(quantity, channel of the block, sum); then, times what it returns, over each group's
    // channels and the cluster's CTAs to joined[slot + quantity].
    template <int Q, typename F> __device__ __forceinline__ void sum(const W (&v)[Q][V], int slot, unsigned block_groups, F each) const {
        const int wide = across * V;
        __syncthreads();
        if (active)
#pragma unroll
            for (int q = 0; q < Q; ++q)
#pragma unroll
                for (int e = 0; e < V; ++e) scratch[(q * deep + ty) * wide + tx * V + e] = v[q][e];
        __syncthreads();
        for (int i = threadIdx.x; i < Q * wide; i += blockDim.x) {
            const int q = i >= wide ? 1 : 0, c = i - q * wide;
            W all = 0;
#pragma unroll 4
            for (int d = 0; d < deep; ++d) all += scratch[(q * deep + d) * wide + c];
            scratch[q * deep * wide + c] = each(q, c, all);  // the first row's place: only this thread reads it
        }
        __syncthreads();
        const int warps = blockDim.x / 32;
        for (int i = threadIdx.x / 32; i < Q * groups; i += warps) {
            const int q = i >= groups ? 1 : 0, g = i - q * groups;
            W all = 0;
            for (int d = threadIdx.x % 32; d < width; d += 32) all += scratch[q * deep * wide + g * width + d];
            for (int o = 16; o; o >>= 1) all += __shfl_xor_sync(~0u, all, o);
            if (threadIdx.x % 32 == 0) total[(slot + q) * block_groups + g] = all;
        }
        if (ranks > 1) cluster_sync();
        else __syncthreads();
        for (int i = threadIdx.x; i < Q * groups; i += blockDim.x) {
            const int q = i >= groups ? 1 : 0, to = (slot + q) * (int)block_groups + i - q * groups;
            W all = total[to];
            if (ranks > 1) {
                all = 0;
                for (uint32_t r = 0; r < ranks; ++r) {
                    W other;
                    cluster_read(other, smem_addr(total + to), r);
                    all += other;
                }
            }
            joined[to] = all;
        }
        __syncthreads();
    }
    // Rows that the cluster's r-th CTA holds.
    __device__ __forceinline__ uint64_t rows_of(uint32_t r, const NormParams<T> &p) const {
        const uint64_t from = (uint64_t)r * p.plan.slab_rows;
        return from < p.positions ? min((uint64_t)p.plan.slab_rows, p.positions - from) : 0;
    }
    // Each thread's (mean, sum of squares about it) of its rows of each channel, joined over the rows'
    // threads, each group's channels and the cluster's CTAs to joined[g] (mean) and joined[block_groups + g]
    // (variance); squares are always about the joint means.  U: units per thread, its channels one by one, or
    // (1) all of them together where they are in one group.
    template <int U> __device__ __forceinline__ void moments(W (&mean)[V], W (&square)[V], const NormParams<T> &p) const {
        constexpr int C = V / U;  // channels per unit
        const int wide = across * U, long_group = width / C;
        const unsigned bg = p.plan.block_groups;
        // the first `longer` threads of a column have one row more than the others
        const W few = (W)(rows / deep);
        const int longer = rows % deep;
        W *means = scratch, *squares = scratch + deep * wide;
        if (C > 1) {  // every channel has the same number of rows
            W all = 0, spread = 0;
#pragma unroll
            for (int e = 0; e < V; ++e) all += mean[e];
            all *= W(1) / W(C);
#pragma unroll
            for (int e = 0; e < V; ++e) spread += square[e] + (ty < longer ? few + W(1) : few) * (mean[e] - all) * (mean[e] - all);
            mean[0] = all, square[0] = spread;
        }
        if (active)
#pragma unroll
            for (int u = 0; u < U; ++u) means[ty * wide + tx * U + u] = mean[u], squares[ty * wide + tx * U + u] = square[u];
        __syncthreads();
        // With a unit per channel, first a thread per channel and part of the rows' threads.
        int levels = deep, each = 1;
        auto rows_in = [&](int level) {  // rows of a level's threads
            const int from = min(deep, level * each), to = min(deep, from + each);
            return (W)(to - from) * few + (W)(min(to, longer) - min(from, longer));
        };
        if (C == 1) {
            levels = max(1, min(deep, (int)blockDim.x / wide)), each = (deep + levels - 1) / levels;
            // Behind the threads' own shares, at most blockDim.x of each; a single part per channel takes the place
            // of the channel's first share, which only its own thread reads.
            W *part_mean = levels > 1 ? scratch + 2 * deep * wide : means;
            W *part_square = levels > 1 ? part_mean + levels * wide : squares;
            for (int i = threadIdx.x; i < levels * wide; i += blockDim.x) {
                const int part = i / wide, c = i - part * wide, from = min(deep, part * each), to = min(deep, from + each);
                const W n = rows_in(part);
                W all = 0, spread = 0;
#pragma unroll 4
                for (int d = from; d < to; ++d) all += (d < longer ? few + W(1) : few) * means[d * wide + c];
                if (n > W(0)) all /= n;
#pragma unroll 4
                for (int d = from; d < to; ++d) {
                    const W off = means[d * wide + c] - all, m = d < longer ? few + W(1) : few;
                    if (m > W(0)) spread += squares[d * wide + c] + m * off * off;
                }
                part_mean[i] = all, part_square[i] = spread;
            }
            means = part_mean, squares = part_square;
            __syncthreads();
        }
        // Then a warp per group over its levels x units, 32 at a time.
        const int lane = threadIdx.x % 32, down = 32 / long_group, right = 32 % long_group;
        for (int g = threadIdx.x / 32; g < groups; g += blockDim.x / 32) {
            const W *gm = means + g * long_group, *gs = squares + g * long_group;
            W all = 0, spread = 0;
            for (int level = lane / long_group, i = lane % long_group; level < levels;) {
                const W n = rows_in(level);
                if (n > W(0)) all += n * gm[level * wide + i];
                level += down, i += right;
                if (i >= long_group) i -= long_group, ++level;
            }
            for (int o = 16; o; o >>= 1) all += __shfl_xor_sync(~0u, all, o);
            if (rows) all /= (W)rows * (W)long_group;
            for (int level = lane / long_group, i = lane % long_group; level < levels;) {
                const W n = rows_in(level), off = gm[level * wide + i] - all;
                if (n > W(0)) spread += gs[level * wide + i] + W(C) * n * off * off;
                level += down, i += right;
                if (i >= long_group) i -= long_group, ++level;
            }
            for (int o = 16; o; o >>= 1) spread += __shfl_xor_sync(~0u, spread, o);
            if (lane == 0) total[g] = all, total[bg + g] = spread;
        }
        if (ranks > 1) cluster_sync();
        else __syncthreads();
        const W inverse = W(1) / (W)p.positions;
        for (int g = threadIdx.x; g < groups; g += blockDim.x) {
            W all = total[g], spread = total[bg + g];
            if (ranks > 1) {
                all = 0, spread = 0;
                for (uint32_t r = 0; r < ranks; ++r) {
                    W other;
                    cluster_read(other, smem_addr(total + g), r);
                    all += (W)rows_of(r, p) * other;
                }
                all *= inverse;
                for (uint32_t r = 0; r < ranks; ++r) {
                    W other, more;
                    cluster_read(other, smem_addr(total + g), r);
                    cluster_read(more, smem_addr(total + bg + g), r);
                    other -= all;
                    spread += more + (W)rows_of(r, p) * (W)width * other * other;
                }
            }
            joined[g] = all, joined[bg + g] = spread * inverse / (W)width;
        }
        __syncthreads();
    }
    // a quantity's joint sum for each channel of this thread's access
    __device__ __forceinline__ void sums_of(int slot, unsigned block_groups, W (&v)[V]) const {
        int g = tx * V / width, left = (g + 1) * width - tx * V;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            v[e] = joined[slot * block_groups + g];
            if (--left == 0) ++g, left = width;
        }
    }
};

template <typename T, int V> __global__ void __launch_bounds__(512, sizeof(WideOf<T>) == 8 ? 1 : 2) norm_slab_kernel(const NormParams<T> p) {
    using W = WideOf<T>;
    in_stream_order();
    if (!chain_admits(p.guard)) return;  // the same answer in every CTA of the grid
    extern __shared__ __align__(16) unsigned char smem[];
    Slab<T, V, 1> at;
    at.place(p, smem);
    const uint64_t c = at.channel();
    const unsigned bg = p.plan.block_groups;
    W mean[V], r[V];
    const int step = at.step();
    at.bring(0, p.x);
    asm volatile("cp.async.wait_all;" ::: "memory");
    const T *row = at.mine[0];
    row_moments<V, false>(at.active && at.ty < at.rows ? (at.rows - at.ty - 1) / at.deep + 1 : 0, [&](W (&x)[V]) {
        at.read(row, x);
        row += step;
    }, mean, r);
    if (at.width % V == 0) at.template moments<1>(mean, r, p);
    else at.template moments<V>(mean, r, p);
    if (at.ranks > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");  // read; see the end
    if (at.rank == 0)
        for (int g = threadIdx.x; g < at.groups; g += blockDim.x) {
            W *to = p.stats_out + 2 * (at.n * p.groups + at.c0 / p.width + g);
            to[0] = at.joined[g];
            to[1] = root(at.joined[bg + g], p.eps);
        }
    if (at.active) {
        W w[V], b[V], x[V];
        parameters<V>(p.weight, c, W(1), w), parameters<V>(p.bias, c, W(0), b);
        at.sums_of(0, bg, mean), at.sums_of(1, bg, r);
#pragma unroll
        for (int e = 0; e < V; ++e) w[e] *= root(r[e], p.eps);
        const T *from = at.mine[0];
        T *to = p.out.at(at.n, at.s0 + at.ty, c);
        const uint64_t stride = at.deep * p.out.row;
        for (int i = at.ty; i < at.rows; i += at.deep, from += step, to += stride) {
            at.read(from, x);
#pragma unroll
            for (int e = 0; e < V; ++e) x[e] = (x[e] - mean[e]) * w[e] + b[e];
            activate<V>(p.activation, x);
            put<T, V>(to, x, p.status, [&] { return (at.n * p.positions + at.s0 + i) * p.channels + c; });
        }
    }
    __syncwarp();
    // the other CTAs may still read this one's sums
    if (at.ranks > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
}

template <typename T, int V> __global__ void __launch_bounds__(512) norm_slab_backward_kernel(const NormParams<T> p) {
    using W = WideOf<T>;
    in_stream_order();
    if (!chain_admits(p.guard)) return;  // the same answer in every CTA of the grid
    extern __shared__ __align__(16) unsigned char smem[];
    Slab<T, V, 2> at;
    at.place(p, smem);
    at.bring(0, p.x);
    at.bring(1, p.dy);
    const uint64_t c = at.channel();
    const unsigned bg = p.plan.block_groups;
    W w[V], b[V], mean[V], r[V], sums[2][V] = {}, x[V], dy[V], h[V], dz[V];
    if (at.active) {
        parameters<V>(p.weight, c, W(1), w), parameters<V>(p.bias, c, W(0), b);
        const W *st = p.stats + 2 * (at.n * p.groups + c / p.width);
        int left = (int)(p.width - c % p.width);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            mean[e] = st[0], r[e] = st[1];
            if (--left == 0 && e + 1 < V) st += 2, left = at.width;
        }
    }
    const W inverse = W(1) / ((W)p.positions * (W)p.width);
    const int step = at.step();
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (at.active) {
        const T *from = at.mine[0], *up = at.mine[1];
        for (int i = at.ty; i < at.rows; i += at.deep, from += step, up += step) {
            at.read(from, x);
            at.read(up, dy);
            bend<V>(p.activation, x, dy, mean, r, w, b, h, dz);
#pragma unroll
            for (int e = 0; e < V; ++e) sums[0][e] += dz[e] * h[e], sums[1][e] += dz[e];
        }
    }
    // c2 and c1 of each group; on the way, this CTA's share of the parameters' gradients
    W *share = p.partial ? p.partial + 2 * (at.n * at.ranks + at.rank) * p.channels + at.c0 : nullptr;
    at.sum(sums, 0, bg, [&](int q, int i, W v) {
        if (share) share[q * p.channels + i] = v;
        return p.weight ? v * p.weight[at.c0 + i] : v;
    });
    if (at.ranks > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");  // read; see the end
    if (at.active) {
        W c1[V], c2[V];
        at.sums_of(0, bg, c2), at.sums_of(1, bg, c1);
#pragma unroll
        for (int e = 0; e < V; ++e) c1[e] *= inverse, c2[e] *= inverse;
        const T *from = at.mine[0], *up = at.mine[1];
        T *to = p.out.at(at.n, at.s0 + at.ty, c);
        const uint64_t stride = at.deep * p.out.row;
        for (int i = at.ty; i < at.rows; i += at.deep, from += step, up += step, to += stride) {
            at.read(from, x);
            at.read(up, dy);
            bend<V>(p.activation, x, dy, mean, r, w, b, h, dz);
#pragma unroll
            for (int e = 0; e < V; ++e) x[e] = r[e] * (dz[e] * w[e] - c1[e] - h[e] * c2[e]);
            put<T, V>(to, x, p.status, [&] { return (at.n * p.positions + at.s0 + i) * p.channels + c; });
        }
    }
    __syncwarp();
    // the other CTAs may still read this one's sums
    if (at.ranks > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
}

// ---- stream form
template <typename T, int V> struct Stream {
    uint64_t n, s0, s1, c;
    int across, deep, tx, ty;
    unsigned chunk;
    bool active;
    __device__ __forceinline__ Stream(const NormParams<T> &p) {
        const NormPlan &plan = p.plan;
        chunk = blockIdx.x % plan.chunks;
        const unsigned tile = blockIdx.x / plan.chunks % plan.tiles;
        n = blockIdx.x / plan.chunks / plan.tiles;
        const uint64_t first = (uint64_t)tile * plan.tile, all = p.channels / V;
        across = (int)min((uint64_t)plan.tile, all - first);
        deep = (int)blockDim.x / across;
        tx = (int)threadIdx.x % across;
        ty = (int)threadIdx.x / across;
        active = ty < deep;
        c = (first + tx) * V;
        s0 = chunk * plan.chunk_rows;
        s1 = min(p.positions, s0 + plan.chunk_rows);
    }
};

// (mean, sum of squares about it) of each channel over a chunk's rows: partial[n][chunk][channel][2].
template <typename T, int V> __global__ void __launch_bounds__(kNormThreads) norm_stream_stats_kernel(const NormParams<T> p) {
    using W = WideOf<T>;
    in_stream_order();
    if (!chain_admits(p.guard)) return;
    __shared__ W means[kNormThreads * V], squares[kNormThreads * V];
    const Stream<T, V> at(p);
    W mean[V], square[V];
    const T *from = p.x.at(at.n, at.s0 + at.ty, at.c);
    const uint64_t stride = at.deep * p.x.row;
    const int count = at.active && at.s0 + at.ty < at.s1 ? (int)((at.s1 - at.s0 - at.ty - 1) / at.deep + 1) : 0;
    row_moments<V, true>(count, [&](W (&x)[V]) {
        Access<T, V>::load(from).open(x);
        from += stride;
    }, mean, square);
#pragma unroll
    for (int e = 0; e < V; ++e) means[threadIdx.x * V + e] = mean[e], squares[threadIdx.x * V + e] = square[e];
    __syncthreads();
    const uint64_t rows = at.s1 - at.s0;
    for (int i = threadIdx.x; i < at.across * V; i += kNormThreads) {
        W mean = 0, all = 0;
        for (int d = 0; d < at.deep; ++d) {
            const W here = (W)((rows + at.deep - 1 - d) / at.deep);  // rows of the d-th thread
            mean += here * means[d * at.across * V + i];
        }
        mean /= (W)rows;
        for (int d = 0; d < at.deep; ++d) {
            const W here = (W)((rows + at.deep - 1 - d) / at.deep), off = means[d * at.across * V + i] - mean;
            if (here > W(0)) all += squares[d * at.across * V + i] + here * off * off;
        }
        const uint64_t channel = at.c - (uint64_t)at.tx * V + i;
        W *to = p.partial + 2 * ((at.n * p.plan.chunks + at.chunk) * p.channels + channel);
        to[0] = mean, to[1] = all;
    }
}

template <typename W> __device__ __forceinline__ W norm_block_sum(W v, W *scratch) {
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    __syncthreads();
    if (threadIdx.x % 32 == 0) scratch[threadIdx.x / 32] = v;
    __syncthreads();
    v = scratch[0];
    for (int i = 1; i < kNormThreads / 32; ++i) v += scratch[i];
    return v;
}

// One CTA per (n, g): the group's statistics from its chunks'.  Also what a call without positions gets.
template <typename T> __global__ void __launch_bounds__(kNormThreads) norm_join_stats_kernel(const NormParams<T> p) {
    using W = WideOf<T>;
    in_stream_order();
    if (!chain_admits(p.guard)) return;
    __shared__ W scratch[kNormThreads / 32];
    const uint64_t n = blockIdx.x / p.groups, g = blockIdx.x % p.groups, parts = p.plan.chunks * p.width;
    const W inverse = p.positions ? W(1) / ((W)p.positions * (W)p.width) : W(0);
    W mean = 0, square = 0;
    if (p.positions) {
        auto part = [&](uint64_t i, W &count) {
            const uint64_t chunk = i / p.width;
            count = (W)(min(p.positions, (chunk + 1) * p.plan.chunk_rows) - chunk * p.plan.chunk_rows);
            return p.partial + 2 * ((n * p.plan.chunks + chunk) * p.channels + g * p.width + i % p.width);
        };
        W count;
        for (uint64_t i = threadIdx.x; i < parts; i += kNormThreads) {
            const W *from = part(i, count);
            mean += count * from[0];
        }
        mean = norm_block_sum(mean, scratch) * inverse;
        for (uint64_t i = threadIdx.x; i < parts; i += kNormThreads) {
            const W *from = part(i, count);
            square += from[1] + count * (from[0] - mean) * (from[0] - mean);
        }
        square = norm_block_sum(square, scratch);
    }
    if (threadIdx.x == 0) {
        p.stats_out[2 * blockIdx.x] = mean;
        p.stats_out[2 * blockIdx.x + 1] = root(square * inverse, p.eps);
    }
}

template <typename T, int V> __global__ void __launch_bounds__(kNormThreads) norm_stream_apply_kernel(const NormParams<T> p) {
    using W = WideOf<T>;
    in_stream_order();
    if (!chain_admits(p.guard)) return;
    const Stream<T, V> at(p);
    if (!at.active) return;
    W w[V], b[V], mean[V], r[V], x[V];
    parameters<V>(p.weight, at.c, W(1), w), parameters<V>(p.bias, at.c, W(0), b);
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const W *st = p.stats + 2 * (at.n * p.groups + (at.c + e) / p.width);
        mean[e] = st[0], r[e] = st[1];
    }
    for (uint64_t s = at.s0 + at.ty; s < at.s1; s += at.deep) {
        Access<T, V>::load(p.x.at(at.n, s, at.c)).open(x);
#pragma unroll
        for (int e = 0; e < V; ++e) x[e] = (x[e] - mean[e]) * r[e] * w[e] + b[e];
        activate<V>(p.activation, x);
        put<T, V>(p.out.at(at.n, s, at.c), x, p.status, [&] { return (at.n * p.positions + s) * p.channels + at.c; });
    }
}

// Sums of dz h and dz of each channel over a chunk's rows: partial[n][chunk][2][channel].
template <typename T, int V> __global__ void __launch_bounds__(kNormThreads) norm_stream_sums_kernel(const NormParams<T> p) {
    using W = WideOf<T>;
    in_stream_order();
    if (!chain_admits(p.guard)) return;
    __shared__ W scratch[kNormThreads * V];
    const Stream<T, V> at(p);
    W dw[V] = {}, db[V] = {};
    if (at.active) {
        W w[V], b[V], mean[V], r[V], x[V], dy[V], h[V], dz[V];
        parameters<V>(p.weight, at.c, W(1), w), parameters<V>(p.bias, at.c, W(0), b);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const W *st = p.stats + 2 * (at.n * p.groups + (at.c + e) / p.width);
            mean[e] = st[0], r[e] = st[1];
        }
        for (uint64_t s = at.s0 + at.ty; s < at.s1; s += at.deep) {
            Access<T, V>::load(p.x.at(at.n, s, at.c)).open(x);
            Access<T, V>::load(p.dy.at(at.n, s, at.c)).open(dy);
            bend<V>(p.activation, x, dy, mean, r, w, b, h, dz);
#pragma unroll
            for (int e = 0; e < V; ++e) dw[e] += dz[e] * h[e], db[e] += dz[e];
        }
    }
    W *to = p.partial + 2 * (at.n * p.plan.chunks + at.chunk) * p.channels + (at.c - (uint64_t)at.tx * V);
    for (int q = 0; q < 2; ++q) {
        __syncthreads();
        if (at.active)
#pragma unroll
            for (int e = 0; e < V; ++e) scratch[threadIdx.x * V + e] = q ? db[e] : dw[e];
        __syncthreads();
        for (int i = threadIdx.x; i < at.across * V; i += kNormThreads) {
            W sum = 0;
            for (int d = 0; d < at.deep; ++d) sum += scratch[d * at.across * V + i];
            to[q * p.channels + i] = sum;
        }
    }
}

// One CTA per (n, g): c1 and c2 from its channels' sums.
template <typename T> __global__ void __launch_bounds__(kNormThreads) norm_join_sums_kernel(const NormParams<T> p) {
    using W = WideOf<T>;
    in_stream_order();
    if (!chain_admits(p.guard)) return;
    __shared__ W scratch[kNormThreads / 32];
    const uint64_t n = blockIdx.x / p.groups, g = blockIdx.x % p.groups;
    W c1 = 0, c2 = 0;
    for (uint64_t i = threadIdx.x; i < p.plan.chunks * p.width; i += kNormThreads) {
        const uint64_t c = g * p.width + i % p.width;
        const W *from = p.partial + 2 * (n * p.plan.chunks + i / p.width) * p.channels + c;
        const W w = p.weight ? p.weight[c] : W(1);
        c2 += w * from[0];
        c1 += w * from[p.channels];
    }
    c1 = norm_block_sum(c1, scratch);
    c2 = norm_block_sum(c2, scratch);
    const W inverse = W(1) / ((W)p.positions * (W)p.width);
    if (threadIdx.x == 0) p.sums[2 * blockIdx.x] = c1 * inverse, p.sums[2 * blockIdx.x + 1] = c2 * inverse;
}

template <typename T, int V> __global__ void __launch_bounds__(kNormThreads) norm_stream_gradient_kernel(const NormParams<T> p) {
    using W = WideOf<T>;
    in_stream_order();
    if (!chain_admits(p.guard)) return;
    const Stream<T, V> at(p);
    if (!at.active) return;
    W w[V], b[V], mean[V], r[V], c1[V], c2[V], x[V], dy[V], h[V], dz[V];
    parameters<V>(p.weight, at.c, W(1), w), parameters<V>(p.bias, at.c, W(0), b);
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const uint64_t st = 2 * (at.n * p.groups + (at.c + e) / p.width);
        mean[e] = p.stats[st], r[e] = p.stats[st + 1], c1[e] = p.sums[st], c2[e] = p.sums[st + 1];
    }
    for (uint64_t s = at.s0 + at.ty; s < at.s1; s += at.deep) {
        Access<T, V>::load(p.x.at(at.n, s, at.c)).open(x);
        Access<T, V>::load(p.dy.at(at.n, s, at.c)).open(dy);
        bend<V>(p.activation, x, dy, mean, r, w, b, h, dz);
#pragma unroll
        for (int e = 0; e < V; ++e) x[e] = r[e] * (dz[e] * w[e] - c1[e] - h[e] * c2[e]);
        put<T, V>(p.out.at(at.n, s, at.c), x, p.status, [&] { return (at.n * p.positions + s) * p.channels + at.c; });
    }
}

// ---- the parameters' gradients from partial sums [rows][2][channels], in a fixed order:
// 32 channels by 32 threads each per CTA
template <typename T> __global__ void __launch_bounds__(1024) norm_parameters_kernel(const NormParams<T> p) {
    using W = WideOf<T>;
    in_stream_order();
    if (!chain_admits(p.guard)) return;
    __shared__ W scratch[2][32][33];
    const uint64_t c = (uint64_t)blockIdx.x * 32 + threadIdx.x % 32;
    const uint64_t rows = p.batch * p.positions ? p.plan.partial_rows : 0;
    W dw = 0, db = 0;
    if (c < p.channels) {
        const W *at = p.partial + c + 2 * p.channels * (threadIdx.x / 32);
#pragma unroll 8
        for (uint64_t i = threadIdx.x / 32; i < rows; i += 32, at += 64 * p.channels) dw += at[0], db += at[p.channels];
    }
    scratch[0][threadIdx.x / 32][threadIdx.x % 32] = dw;
    scratch[1][threadIdx.x / 32][threadIdx.x % 32] = db;
    __syncthreads();
    const int which = threadIdx.x / 32, lane = threadIdx.x % 32;  // a warp per channel
    dw = scratch[0][lane][which], db = scratch[1][lane][which];
    for (int o = 16; o; o >>= 1) dw += __shfl_xor_sync(~0u, dw, o), db += __shfl_xor_sync(~0u, db, o);
    const uint64_t channel = (uint64_t)blockIdx.x * 32 + which;
    if (lane != 0 || channel >= p.channels) return;
    const uint64_t first = p.batch * p.positions * p.channels + channel;
    if (p.dweight) {
        p.dweight[channel] = dw;
        if (const unsigned kind = result_kind(dw)) record_fault(p.status, first, kind);
    }
    if (p.dbias) {
        p.dbias[channel] = db;
        if (const unsigned kind = result_kind(db)) record_fault(p.status, first + p.channels, kind);
    }
}

}  // namespace pcu

using namespace pcu;

namespace {

// What the two calls and their guarded forms pass on.
struct NormCall {
    int dtype, activation;
    const void *input, *upstream, *weight, *bias, *stats_in;
    void *out, *stats_out, *dweight, *dbias;
    uint64_t batch, positions, channels, groups;
    uint64_t input_batch_stride, input_stride, upstream_batch_stride, upstream_stride, out_batch_stride, out_stride;
    uint32_t eps_bits;
    bool backward;
    void *workspace;
    size_t workspace_bytes;
    uint64_t *status;
    void *stream;
};

constexpr uint64_t kMost = 1ull << 56;  // elements, and elements that strides span: addresses stay in 64 bits

bool shape_fits(uint64_t batch, uint64_t positions, uint64_t channels, uint64_t groups) {
    return channels <= (1ull << 30) && positions <= (1ull << 40) &&
           pcu_host::multiply_fits(batch, groups, 0x7fffffffull) && pcu_host::multiply_fits(positions, channels, kMost) &&
           pcu_host::multiply_fits(positions * channels, batch, kMost);
}

constexpr size_t kSlabMost = 200 * 1024;  // shared memory of a CTA for a slab

// `vector`: elements per access, 16 bytes' worth or 1.  `near`: samples span less than 2^31 elements.  No
// extent is 0.
NormPlan plan_norm(int dtype, int vector, bool near, uint64_t batch, uint64_t positions, uint64_t channels, uint64_t groups,
                   bool backward) {
    NormPlan p{};
    const uint64_t width = channels / groups, bytes = pcu_host::element_bytes(dtype), wide = dtype == PCU_B200_F64 ? 8 : 4;
    const uint64_t sms = (uint64_t)pcu_host::sm_count();
    p.vector = vector;
    // Warp form: 16 elements of a lane are in registers (and as many of dy, and four parameters' worth), so
    // a group has at most 512 of them.
    if (near && width % vector == 0 && positions <= 512 && positions * (width / vector) * vector <= 512) {
        p.form = NormPlan::kWarp;
        p.items = (unsigned)(positions * (width / vector));
        // A lane takes two accesses (one backward), or 8 single elements (4), where the group has them: fewer
        // lanes join their sums in fewer steps (8192 x 4096, groups of 128, F32: 51 us against 54 with four and 58 with
        // one; backward one holds the registers of two loads in flight, two do not: 99 against 112 us).
        const unsigned accesses = vector == 1 ? (backward ? 4 : 8) : (backward ? 1 : 2);
        p.lanes = 1;
        while (p.lanes < 32 && (unsigned)p.lanes * accesses < p.items) p.lanes *= 2;
        p.per_lane = (int)((p.items + p.lanes - 1) / p.lanes);
        const uint64_t per = 32 / p.lanes, sets = (groups + per - 1) / per;
        const uint64_t ctas = p.per_lane > 4 ? 1 : warp_form_ctas((int)(vector * p.per_lane * wide), backward);
        // Each warp walks over a slice of the batch; as many warps as are resident at once.
        p.slices = (unsigned)std::max<uint64_t>(1, std::min<uint64_t>(batch, sms * ctas * (kNormThreads / 32) / sets));
        p.partial_rows = p.slices;
        p.workspace = backward ? 2 * p.partial_rows * channels : 0;
        return p;
    }
    // Slab form: blocks of whole groups whose rows are at least 128 bytes and whole accesses, in the
    // smallest cluster whose CTAs hold at most 84 KB, so that two share an SM and overlap loading, sums and stores
    // while their threads have some ten rows each to earn their set-up (48 KB: 158 against 131 us at 16 x
    // 4095 x 1280 BF16 forward, 164 against 122 us at 32 x 1024 x 1280 backward), or 200 KB in a cluster of 8;
    // more CTAs, down to 16 KB each, when they do not fill the SMs twice.
    const uint64_t most = 84 * 1024;
    const uint64_t tensors = backward ? 2 : 1;
    const uint64_t step = (uint64_t)vector / std::gcd(width, (uint64_t)vector);
    auto try_slab = [&](uint64_t block) {
        block = std::min(block, groups);
        const uint64_t across = block * width / vector;
        if (across > 512 || block * width % vector != 0) return false;
        const uint64_t row = block * width * bytes * tensors;
        const uint64_t blocks = (groups + block - 1) / block, clusters = batch * blocks;
        uint64_t ranks = 1;
        while (ranks < 8 && (positions + ranks - 1) / ranks * row > most) ranks *= 2;
        while (ranks < 8 && clusters * ranks < 2 * sms && (positions + ranks - 1) / ranks * row > 16384) ranks *= 2;
        // The SMs come in 8 groups, and a cluster stays within one.  Where so many clusters take two turns, but
        // somewhat smaller ones a single turn, those are taken (20 clusters at 5 x 4095 x 320: of 8 CTAs 18.6 us, of 6
        // 16.7 us).
        auto turns = [&](uint64_t r) { return (clusters + 8 * (sms / 8 / r) - 1) / (8 * (sms / 8 / r)); };
        if (sms >= 64 && turns(ranks) == 2)
            for (uint64_t r = ranks - 1; 2 * r > ranks; --r)
                if (turns(r) == 1 && (positions + r - 1) / r * row <= 128 * 1024) {
                    ranks = r;
                    break;
                }
        const uint64_t rows = (positions + ranks - 1) / ranks;
        const uint64_t threads = across > 256 ? 512 : 256;
        const uint64_t extra = 2 * threads * (vector + 1) * wide + 4 * block * wide + 64;
        if (rows > 0x7fffffffull || rows * row + extra + 64 > kSlabMost || batch * blocks * ranks > 0x7fffffffull) return false;
        p.form = NormPlan::kSlab;
        p.block_groups = (unsigned)block;
        p.blocks = (unsigned)blocks;
        p.ranks = (unsigned)ranks;
        p.threads = (unsigned)threads;
        p.slab_rows = (unsigned)rows;
        p.slab_bytes = (rows * block * width * bytes + 15) / 16 * 16;
        p.shared = tensors * p.slab_bytes + extra;
        p.partial_rows = batch * ranks;
        p.workspace = backward ? 2 * p.partial_rows * channels : 0;
        return true;
    };
    const uint64_t need = (128 + width * bytes - 1) / (width * bytes);
    const uint64_t block = (need + step - 1) / step * step;
    if (try_slab(block) || (block > step && try_slab(step))) return p;
    // Stream form: column tiles of a CTA's threads, row chunks to fill the SMs four times.
    p.form = NormPlan::kStream;
    const uint64_t across = channels / vector;
    p.tile = (unsigned)std::min<uint64_t>(across, kNormThreads);
    p.tiles = (unsigned)((across + p.tile - 1) / p.tile);
    const uint64_t deep = kNormThreads / p.tile;
    uint64_t chunks = std::max<uint64_t>(1, std::min<uint64_t>(4 * sms / std::max<uint64_t>(1, batch * p.tiles),
                                                               (positions + 4 * deep - 1) / (4 * deep)));
    p.chunk_rows = (positions + chunks - 1) / chunks;
    p.chunks = (unsigned)((positions + p.chunk_rows - 1) / p.chunk_rows);
    p.partial_rows = batch * p.chunks;
    p.workspace = 2 * p.partial_rows * channels + (backward ? 2 * batch * groups : 0);
    return p;
}

// 0 for what the calls refuse.  Enough for either access width.
size_t workspace_size(int dtype, uint64_t batch, uint64_t positions, uint64_t channels, uint64_t groups, bool backward) {
    const size_t bytes = pcu_host::element_bytes(dtype);
    if (!bytes || groups == 0 || channels % groups != 0 || !shape_fits(batch, positions, channels, groups)) return 0;
    if (batch == 0 || positions == 0 || channels == 0) return 0;
    uint64_t need = 0;  // for either access width, samples near and far
    const int vector = (int)(16 / bytes);
    for (const bool near : {true, false}) {
        need = std::max(need, plan_norm(dtype, 1, near, batch, positions, channels, groups, backward).workspace);
        if (channels % vector == 0)
            need = std::max(need, plan_norm(dtype, vector, near, batch, positions, channels, groups, backward).workspace);
    }
    return need * (dtype == PCU_B200_F64 ? 8 : 4);
}

#define PCU_LAUNCHED(call)               \
    do {                                 \
        rc = call;                       \
        if (rc) return rc;               \
        p.guard = chain_follow(p.guard); \
    } while (0)

template <typename T, int V, int K> int run_warp(NormParams<T> p, bool backward, cudaStream_t stream) {
    constexpr int U = std::max(1, 16 / (V * K)), UB = std::max(1, 8 / (V * K));
    const uint64_t per = 32 / p.plan.lanes, warps = (p.groups + per - 1) / per * p.plan.slices;
    const unsigned blocks = (unsigned)((warps + kNormThreads / 32 - 1) / (kNormThreads / 32));
    if (backward) return pcu_host::launch_grid(norm_warp_backward_kernel<T, V, K, UB>, blocks, kNormThreads, stream, p);
    return pcu_host::launch_grid(norm_warp_kernel<T, V, K, U>, blocks, kNormThreads, stream, p);
}

template <typename T, int V> int run_norm(NormParams<T> p, bool backward, cudaStream_t stream) {
    int rc = PCU_B200_OK;
    const NormPlan &plan = p.plan;
    if (plan.form == NormPlan::kWarp) {
        // accesses per lane: 1, 2, 4, or what 16 elements make
        if (plan.per_lane == 1) rc = run_warp<T, V, 1>(p, backward, stream);
        else if (plan.per_lane == 2) rc = run_warp<T, V, 2>(p, backward, stream);
        else if (plan.per_lane <= 4) rc = run_warp<T, V, std::min(4, 16 / V)>(p, backward, stream);
        else rc = run_warp<T, V, 16 / V>(p, backward, stream);
        if (rc) return rc;
        p.guard = chain_follow(p.guard);
    } else if (plan.form == NormPlan::kSlab) {
        const unsigned grid = (unsigned)(p.batch * plan.blocks * plan.ranks);
        if (backward) {
            if ((rc = pcu_host::allow_shared<norm_slab_backward_kernel<T, V>>((int)kSlabMost))) return rc;
            rc = pcu_host::launch_cluster(norm_slab_backward_kernel<T, V>, grid, plan.threads, plan.shared, plan.ranks, stream, p);
        } else {
            if ((rc = pcu_host::allow_shared<norm_slab_kernel<T, V>>((int)kSlabMost))) return rc;
            rc = pcu_host::launch_cluster(norm_slab_kernel<T, V>, grid, plan.threads, plan.shared, plan.ranks, stream, p);
        }
        if (rc) return rc;
        p.guard = chain_follow(p.guard);
    } else {
        const unsigned grid = (unsigned)(p.batch * plan.tiles * plan.chunks), groups = (unsigned)(p.batch * p.groups);
        if (backward) {
            PCU_LAUNCHED((pcu_host::launch_grid(norm_stream_sums_kernel<T, V>, grid, kNormThreads, stream, p)));
            PCU_LAUNCHED((pcu_host::launch_grid(norm_join_sums_kernel<T>, groups, kNormThreads, stream, p)));
            PCU_LAUNCHED((pcu_host::launch_grid(norm_stream_gradient_kernel<T, V>, grid, kNormThreads, stream, p)));
        } else {
            PCU_LAUNCHED((pcu_host::launch_grid(norm_stream_stats_kernel<T, V>, grid, kNormThreads, stream, p)));
            PCU_LAUNCHED((pcu_host::launch_grid(norm_join_stats_kernel<T>, groups, kNormThreads, stream, p)));
            PCU_LAUNCHED((pcu_host::launch_grid(norm_stream_apply_kernel<T, V>, grid, kNormThreads, stream, p)));
        }
    }
    return PCU_B200_OK;
}

template <typename T> int typed_norm(const NormCall &c, const ChainGuard &guard) {
    using W = WideOf<T>;
    constexpr int V = 16 / sizeof(T);
    NormParams<T> p{};
    p.x = {(const T *)c.input, c.input_batch_stride, c.input_stride};
    p.dy = {(const T *)c.upstream, c.upstream_batch_stride, c.upstream_stride};
    p.out = {(T *)c.out, c.out_batch_stride, c.out_stride};
    p.weight = (const W *)c.weight;
    p.bias = (const W *)c.bias;
    p.stats_out = (W *)c.stats_out;
    p.stats = c.backward ? (const W *)c.stats_in : (const W *)c.stats_out;
    p.dweight = (W *)c.dweight;
    p.dbias = (W *)c.dbias;
    p.batch = c.batch;
    p.positions = c.positions;
    p.channels = c.channels;
    p.groups = c.groups;
    p.width = c.channels / c.groups;
    p.eps = (W)pcu_host::rate_f32(c.eps_bits);
    p.activation = c.activation;
    p.status = reinterpret_cast<unsigned long long *>(c.status);
    p.guard = guard;
    cudaStream_t stream = pcu_host::as_stream(c.stream);
    int rc = PCU_B200_OK;
    if (c.batch && c.positions) {
        // 16-byte accesses where every row of every tensor starts on 16 bytes and ends with whole ones
        auto whole = [&](const void *base, uint64_t batch_stride, uint64_t stride) {
            return pcu_host::aligned(base, 16) && (c.batch == 1 || batch_stride % V == 0) &&
                   (c.positions == 1 || stride % V == 0);
        };
        const bool wide = c.channels % V == 0 && whole(c.input, c.input_batch_stride, c.input_stride) &&
                          whole(c.out, c.out_batch_stride, c.out_stride) &&
                          (!c.backward || whole(c.upstream, c.upstream_batch_stride, c.upstream_stride));
        auto spans = [&](uint64_t stride) { return (c.positions - 1) * stride + c.channels < (1ull << 31); };
        const bool near = spans(c.input_stride) && spans(c.out_stride) && (!c.backward || spans(c.upstream_stride));
        p.plan = plan_norm(c.dtype, wide ? V : 1, near, c.batch, c.positions, c.channels, c.groups, c.backward);
        p.partial = (W *)c.workspace;
        p.sums = p.partial + 2 * p.plan.partial_rows * p.channels;  // stream form
        // partial sums are for the stream form's groups, or for gradients that are wanted
        if (c.backward && p.plan.form != NormPlan::kStream && !c.dweight && !c.dbias) p.partial = nullptr;
        if (p.plan.form == NormPlan::kStream &&
            !pcu_host::multiply_fits(c.batch * p.plan.tiles, p.plan.chunks, 0x7fffffffull))
            return PCU_B200_ERROR_SIZE_OVERFLOW;
        rc = wide ? run_norm<T, V>(p, c.backward, stream) : run_norm<T, 1>(p, c.backward, stream);
        if (rc) return rc;
        p.guard = chain_follow(p.guard);
    } else if (!c.backward) {
        return pcu_host::launch_grid(norm_join_stats_kernel<T>, (unsigned)(c.batch * c.groups), kNormThreads, stream, p);
    }
    if (c.backward && (c.dweight || c.dbias)) {
        rc = pcu_host::launch_grid(norm_parameters_kernel<T>, (unsigned)((c.channels + 31) / 32), 1024, stream, p);
    }
    return rc;
}

// Rows of `channels` elements that do not overlap: a sample's rows lie within the batch stride, or, with
// positions first, a position's rows within the row stride.
bool good_maps(const void *base, uint64_t batch, uint64_t positions, uint64_t channels, uint64_t batch_stride,
               uint64_t stride) {
    if (!base || (positions > 1 && stride < channels) || (batch > 1 && batch_stride < channels)) return false;
    if (batch <= 1 || positions <= 1) return true;
    return batch_stride >= (positions - 1) * stride + channels || stride >= (batch - 1) * batch_stride + channels;
}

int norm(const NormCall &c, const ChainGuard &guard) {
    if (!pcu_host::element_bytes(c.dtype) || c.activation < 0 || c.activation > PCU_B200_ACTIVATION_GELU || !c.status)
        return PCU_B200_ERROR_INVALID_ARGUMENT;
    if (c.groups == 0 || c.channels % c.groups != 0) return PCU_B200_ERROR_INVALID_ARGUMENT;
    const float eps = pcu_host::rate_f32(c.eps_bits);
    if (!std::isfinite(eps) || std::signbit(eps)) return PCU_B200_ERROR_INVALID_ARGUMENT;
    if (!shape_fits(c.batch, c.positions, c.channels, c.groups) || c.input_batch_stride > kMost || c.input_stride > kMost || c.out_batch_stride > kMost || c.out_stride > kMost ||
        (c.backward && (c.upstream_batch_stride > kMost || c.upstream_stride > kMost)) ||
        !pcu_host::multiply_fits(c.input_batch_stride, c.batch, kMost) ||
        !pcu_host::multiply_fits(c.out_batch_stride, c.batch, kMost) ||
        (c.backward && !pcu_host::multiply_fits(c.upstream_batch_stride, c.batch, kMost)) ||
        !pcu_host::multiply_fits(c.input_stride, c.positions, kMost) ||
        !pcu_host::multiply_fits(c.out_stride, c.positions, kMost) ||
        (c.backward && !pcu_host::multiply_fits(c.upstream_stride, c.positions, kMost)))
        return PCU_B200_ERROR_SIZE_OVERFLOW;
    if (c.channels == 0 || (!c.backward && c.batch == 0) ||
        (c.backward && (c.batch == 0 || c.positions == 0) && !c.dweight && !c.dbias))
        return chain_decide_only(guard, pcu_host::as_stream(c.stream));
    if (!c.backward && !c.stats_out) return PCU_B200_ERROR_INVALID_ARGUMENT;
    const size_t bytes = pcu_host::element_bytes(c.dtype), wide = c.dtype == PCU_B200_F64 ? 8 : 4;
    for (const void *p : {c.input, c.upstream, (const void *)c.out})
        if (!pcu_host::aligned(p, bytes)) return PCU_B200_ERROR_INVALID_ARGUMENT;
    for (const void *p : {c.weight, c.bias, c.stats_in, (const void *)c.stats_out, (const void *)c.dweight, (const void *)c.dbias})
        if (!pcu_host::aligned(p, wide)) return PCU_B200_ERROR_INVALID_ARGUMENT;
    if (!pcu_host::aligned(c.status, 8)) return PCU_B200_ERROR_INVALID_ARGUMENT;
    if (c.batch && c.positions) {
        if (!good_maps(c.input, c.batch, c.positions, c.channels, c.input_batch_stride, c.input_stride) ||
            !good_maps(c.out, c.batch, c.positions, c.channels, c.out_batch_stride, c.out_stride))
            return PCU_B200_ERROR_INVALID_ARGUMENT;
        if (c.backward && (!c.stats_in || !good_maps(c.upstream, c.batch, c.positions, c.channels,
                                                     c.upstream_batch_stride, c.upstream_stride)))
            return PCU_B200_ERROR_INVALID_ARGUMENT;
        // in place means element for element
        auto in_place_ok = [&](const void *base, uint64_t batch_stride, uint64_t stride) {
            return base != c.out || ((c.batch == 1 || batch_stride == c.out_batch_stride) &&
                                     (c.positions == 1 || stride == c.out_stride));
        };
        if (!in_place_ok(c.input, c.input_batch_stride, c.input_stride) ||
            (c.backward && !in_place_ok(c.upstream, c.upstream_batch_stride, c.upstream_stride)))
            return PCU_B200_ERROR_INVALID_ARGUMENT;
        const size_t need = workspace_size(c.dtype, c.batch, c.positions, c.channels, c.groups, c.backward);
        if (need && (!c.workspace || c.workspace_bytes < need || !pcu_host::aligned(c.workspace, 16)))
            return PCU_B200_ERROR_WORKSPACE;
    }
    switch (c.dtype) {
    case PCU_B200_F32: return typed_norm<float>(c, guard);
    case PCU_B200_F64: return typed_norm<double>(c, guard);
    case PCU_B200_F16: return typed_norm<__half>(c, guard);
    default: return typed_norm<__nv_bfloat16>(c, guard);
    }
}

}  // namespace

#define PCU_NORM_SHAPE                                                                                              \
    uint64_t batch, uint64_t positions, uint64_t channels, uint64_t groups, uint64_t input_batch_stride,            \
        uint64_t input_stride
#define PCU_NORM_FORWARD                                                                                            \
    int dtype, int activation, const void *input, const void *weight, const void *bias, void *out, void *stats,     \
        PCU_NORM_SHAPE, uint64_t out_batch_stride, uint64_t out_stride, uint32_t eps_bits_f32, void *workspace,     \
        size_t workspace_bytes
#define PCU_NORM_BACKWARD                                                                                           \
    int dtype, int activation, const void *input, const void *upstream, const void *weight, const void *bias,       \
        const void *stats, void *gradient, void *weight_gradient, void *bias_gradient, PCU_NORM_SHAPE,              \
        uint64_t upstream_batch_stride, uint64_t upstream_stride, uint64_t gradient_batch_stride,                   \
        uint64_t gradient_stride, void *workspace, size_t workspace_bytes

#define PCU_NORM_COMMON(c, status_word)                                                                             \
    c.dtype = dtype;                                                                                                \
    c.activation = activation;                                                                                      \
    c.input = input;                                                                                                \
    c.weight = weight;                                                                                              \
    c.bias = bias;                                                                                                  \
    c.batch = batch;                                                                                                \
    c.positions = positions;                                                                                        \
    c.channels = channels;                                                                                          \
    c.groups = groups;                                                                                              \
    c.input_batch_stride = input_batch_stride;                                                                      \
    c.input_stride = input_stride;                                                                                  \
    c.workspace = workspace;                                                                                        \
    c.workspace_bytes = workspace_bytes;                                                                            \
    c.status = status_word;                                                                                         \
    c.stream = stream

static int forward(PCU_NORM_FORWARD, uint64_t *status, void *stream, const ChainGuard &guard) {
    NormCall c{};
    PCU_NORM_COMMON(c, status);
    c.out = out;
    c.stats_out = stats;
    c.out_batch_stride = out_batch_stride;
    c.out_stride = out_stride;
    c.eps_bits = eps_bits_f32;
    return norm(c, guard);
}

static int backward(PCU_NORM_BACKWARD, uint64_t *status, void *stream, const ChainGuard &guard) {
    NormCall c{};
    PCU_NORM_COMMON(c, status);
    c.backward = true;
    c.upstream = upstream;
    c.stats_in = stats;
    c.out = gradient;
    c.dweight = weight_gradient;
    c.dbias = bias_gradient;
    c.upstream_batch_stride = upstream_batch_stride;
    c.upstream_stride = upstream_stride;
    c.out_batch_stride = gradient_batch_stride;
    c.out_stride = gradient_stride;
    return norm(c, guard);
}

#define PCU_NORM_FORWARD_ARGS                                                                                       \
    dtype, activation, input, weight, bias, out, stats, batch, positions, channels, groups, input_batch_stride,     \
        input_stride, out_batch_stride, out_stride, eps_bits_f32, workspace, workspace_bytes
#define PCU_NORM_BACKWARD_ARGS                                                                                      \
    dtype, activation, input, upstream, weight, bias, stats, gradient, weight_gradient, bias_gradient, batch,       \
        positions, channels, groups, input_batch_stride, input_stride, upstream_batch_stride, upstream_stride,      \
        gradient_batch_stride, gradient_stride, workspace, workspace_bytes

extern "C" size_t pcu_b200_group_norm_workspace_size(int dtype, uint64_t batch, uint64_t positions, uint64_t channels,
                                                     uint64_t groups) {
    return workspace_size(dtype, batch, positions, channels, groups, false);
}

extern "C" size_t pcu_b200_group_norm_backward_workspace_size(int dtype, uint64_t batch, uint64_t positions,
                                                              uint64_t channels, uint64_t groups) {
    return workspace_size(dtype, batch, positions, channels, groups, true);
}

extern "C" int pcu_b200_group_norm(PCU_NORM_FORWARD, uint64_t *status, void *stream) {
    return forward(PCU_NORM_FORWARD_ARGS, status, stream, ChainGuard{});
}

extern "C" int pcu_b200_group_norm_backward(PCU_NORM_BACKWARD, uint64_t *status, void *stream) {
    return backward(PCU_NORM_BACKWARD_ARGS, status, stream, ChainGuard{});
}

extern "C" int pcu_b200_guarded_group_norm(PCU_NORM_FORWARD, uint64_t *chain_records, uint32_t chain_stage,
                                           void *stream) {
    if (!chain_records) return PCU_B200_ERROR_INVALID_ARGUMENT;
    return forward(PCU_NORM_FORWARD_ARGS, chain_records + 2ull * chain_stage, stream,
                   pcu_host::slab_guard(chain_records, chain_stage));
}

extern "C" int pcu_b200_guarded_group_norm_backward(PCU_NORM_BACKWARD, uint64_t *chain_records, uint32_t chain_stage,
                                                    void *stream) {
    if (!chain_records) return PCU_B200_ERROR_INVALID_ARGUMENT;
    return backward(PCU_NORM_BACKWARD_ARGS, chain_records + 2ull * chain_stage, stream,
                    pcu_host::slab_guard(chain_records, chain_stage));
}
