// distill.cu -- distillation loss against a teacher's top logits, and its gradient.
//
// Row i has the student's logits z[0..V), the teacher's entries (idx_j, t_j), j < k, a weight w
// and an upstream gradient u.  With temperature T
//   q = softmax(z / T) over the vocabulary, p = softmax(t / T) over the row's present entries,
//   loss = w T^2 sum_j p_j (ln p_j - ln q[idx_j]),   d loss u / d z_v = u w T (q_v - sum_{idx_j = v} p_j).
// The row statistics are m = max z and s = sum exp((z - m) / T): q_v = exp((z_v - m) / T) / s keeps
// the relative precision of binary32, which a single log-sum-exp of magnitude 50 would not.
#include <type_traits>

#include "learn.cuh"
#include "provider.h"
#include "tma.cuh"

namespace pcu {

constexpr int kDistillThreads = 256;
constexpr int kMostChunks = 14;  // of a slice; 16 KB each

template <typename T> struct DistillParams {
    using W = WideOf<T>;
    const T *logits;
    uint64_t vocab, stride;
    const int64_t *indices;
    const W *top;
    int k;
    const W *weights;
    W temperature, to_log2;  // T and log2(e) / T
    double t_inverse;
    W *loss;                 // null: gradient only
    W *stats_out;            // may be null
    const W *stats_in;       // gradient only
    const W *upstream;       // null: 1
    int upstream_uniform;
    T *gradient;             // null: loss only
    uint64_t gradient_stride;
    int slice;            // elements of a row per CTA of its cluster (whole granules)
    uint32_t slice_bytes;
    int claims;           // places of the table of claimed indices: a power of two, at least 2 k
    unsigned long long *status;
    ChainGuard guard;
};

template <typename V> __device__ __forceinline__ V block_sum(V v, V *scratch) {
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    __syncthreads();
    if (threadIdx.x % 32 == 0) scratch[threadIdx.x / 32] = v;
    __syncthreads();
    v = scratch[0];
    for (int i = 1; i < kDistillThreads / 32; ++i) v += scratch[i];
    return v;
}

template <typename V> __device__ __forceinline__ V block_max(V v, V *scratch) {
    for (int o = 16; o; o >>= 1) v = fmax(v, __shfl_xor_sync(~0u, v, o));
    __syncthreads();
    if (threadIdx.x % 32 == 0) scratch[threadIdx.x / 32] = v;
    __syncthreads();
    v = scratch[0];
    for (int i = 1; i < kDistillThreads / 32; ++i) v = fmax(v, scratch[i]);
    return v;
}

// Rows that no cluster holds: one CTA per row, which it reads twice.
template <typename T> __global__ void __launch_bounds__(kDistillThreads) distill_kernel(const DistillParams<T> p) {
    using W = WideOf<T>;
    in_stream_order();
    if (!chain_admits(p.guard)) return;
    __shared__ double scratch_d[kDistillThreads / 32];
    __shared__ W scratch_w[kDistillThreads / 32];
    __shared__ double prob[PCU_B200_DISTILL_TOP_MAX];
    __shared__ double chosen[PCU_B200_DISTILL_TOP_MAX];
    __shared__ int place[PCU_B200_DISTILL_TOP_MAX];
    const uint64_t row = blockIdx.x;
    const T *z = p.logits + row * p.stride;
    T *g = p.gradient ? p.gradient + row * p.gradient_stride : nullptr;
    const W weight = p.weights ? p.weights[row] : W(1);

    // the teacher's softmax, in binary64 (k values a row)
    double a_max = -INFINITY;
    int bad = 0;
    for (int j = threadIdx.x; j < p.k; j += kDistillThreads) {
        const int64_t at = p.indices[row * p.k + j];
        const double t = (double)p.top[row * p.k + j];
        bool there = at >= 0 && t != -INFINITY;
        if (there && ((uint64_t)at >= p.vocab || !isfinite(t))) {
            bad = 1;
            there = false;
        }
        place[j] = there ? (int)at : -1;
        prob[j] = there ? t : -INFINITY;
        a_max = fmax(a_max, prob[j]);
    }
    a_max = block_max(a_max, scratch_d);
    bad = __syncthreads_or(bad);
    const bool skip = weight == W(0) || (a_max == -INFINITY && !bad);
    if (skip) {  // nothing to learn from
        if (threadIdx.x == 0) {
            if (p.loss) p.loss[row] = W(0);
            if (p.stats_out) p.stats_out[2 * row] = W(0), p.stats_out[2 * row + 1] = W(1);
        }
        if (g)
            for (uint64_t v = threadIdx.x; v < p.vocab; v += kDistillThreads) g[v] = Elem<T>::round(W(0));
        return;
    }
    double mass = 0;
    for (int j = threadIdx.x; j < p.k; j += kDistillThreads)
        if (place[j] >= 0) mass += exp((prob[j] - a_max) * p.t_inverse);
    mass = block_sum(mass, scratch_d);
    const double ln_mass = log(mass);

    W m, s;
    if (p.stats_in) {
        m = p.stats_in[2 * row];
        s = p.stats_in[2 * row + 1];
    } else {
        // running maximum and sum; a logit of -infinity is a masked entry of the vocabulary
        m = -INFINITY;
        s = 0;
        for (uint64_t v = threadIdx.x; v < p.vocab; v += kDistillThreads) {
            const W x = Elem<T>::load(z[v]);
            if (x > m) {
                s = (m == -INFINITY ? W(0) : s * fast_exp2((m - x) * p.to_log2)) + W(1);
                m = x;
            } else if (x != -INFINITY) {
                s += fast_exp2((x - m) * p.to_log2);
            }
        }
        const W all = block_max(m, scratch_w);
        s = block_sum(isnan(s) ? s : (m == -INFINITY ? W(0) : s * fast_exp2((m - all) * p.to_log2)), scratch_w);
        m = all;
        if (threadIdx.x == 0 && p.stats_out) p.stats_out[2 * row] = m, p.stats_out[2 * row + 1] = s;
    }
    const W up = p.upstream ? p.upstream[p.upstream_uniform ? 0 : row] : W(1);
    const bool invalid = bad || !isfinite(m) || !isfinite(s) || !(s > W(0)) || !isfinite(weight) || (g && !isfinite(up));

    double terms = 0;
    for (int j = threadIdx.x; j < p.k; j += kDistillThreads) {
        if (place[j] < 0) continue;
        const double zj = (double)Elem<T>::load(z[place[j]]);
        const double a = (prob[j] - a_max) * p.t_inverse, pj = exp(a) / mass;
        if (pj > 0)
            terms += pj * ((a - ln_mass) - ((zj - (double)m) / (double)p.temperature - log((double)s)));
        chosen[j] = zj;
        prob[j] = pj;
    }
    unsigned kind = invalid ? (unsigned)PCU_B200_KIND_INVALID : 0u;
    if (p.loss) {
        terms = block_sum(terms, scratch_d);
        const W value =
            invalid ? W(NAN) : (W)((double)weight * (double)p.temperature * (double)p.temperature * terms);
        if (threadIdx.x == 0) p.loss[row] = value;
        if (!kind) kind = result_kind(value);
    }
    __syncthreads();
    if (g) {
        const W factor = up * weight * p.temperature;
        const W inverse = W(1) / s;
        unsigned worst = 0;
        for (uint64_t v = threadIdx.x; v < p.vocab; v += kDistillThreads) {
            const W q = fast_exp2((Elem<T>::load(z[v]) - m) * p.to_log2) * inverse;
            const T r = Elem<T>::round(invalid ? W(NAN) : factor * q);
            worst = max(worst, result_kind(Elem<T>::load(r)));
            g[v] = r;
        }
        __syncthreads();
        if (!invalid)
            for (int j = threadIdx.x; j < p.k; j += kDistillThreads) {
                if (place[j] < 0) continue;
                bool first = true;  // the first entry of an index carries the sum of all of them
                for (int i = 0; i < j; ++i) first &= place[i] != place[j];
                if (!first) continue;
                double sum = prob[j];
                for (int i = j + 1; i < p.k; ++i)
                    if (place[i] == place[j]) sum += prob[i];
                const W q = fast_exp2(((W)chosen[j] - m) * p.to_log2) * inverse;
                const T r = Elem<T>::round(factor * (q - (W)sum));
                worst = max(worst, result_kind(Elem<T>::load(r)));
                g[place[j]] = r;
            }
        if (worst && !kind) kind = worst;
    }
    if (kind) record_fault(p.status, row, kind);
}

// ---- rows in shared memory
//
// Measured: a step over 4096 x 131072 BF16 512 us, 4.2 TB/s of the 6.55 that a copy reaches; 777 x 50003 F32 72 us;
// backward alone, 2048 x 32768 BF16, 54 us = 5.0 TB/s; a loss of 4 rows of 131072 6.8 us, mostly the launch.
// What bounds it is each CTA's chain: of some 24,000 cycles 10,000 are spent until the slice has landed and is
// summed, up to 5,000 on joining (warps, cluster, the teacher's exponentials; the loss's own sums follow the gradient),
// 6,500 on the gradient, and three CTAs per SM, all that shared memory holds, cover each other's gaps only in part.
//
// A cluster of 1, 2, 4 or 8 CTAs takes a row, each a slice of the vocabulary that stays in its shared
// memory: bulk copies bring it in once, the running maximum and sum are taken as it lands, the CTAs
// join theirs through the cluster, and the gradient is formed from shared memory.  So a step reads
// the logits once and writes the gradient once, which is what it cannot do without; with the rows
// read a second time through L2, 592 resident rows of 256 KB were more than L2 holds.
// Bulk copies move whole 16-byte granules; a row that starts or ends inside one has its edges copied
// by threads, so any alignment keeps the wide loads.  The slice keeps the row's phase: the byte at
// address a lies at (a - first granule's address).

constexpr int kChunk = 16384;  // bytes per bulk copy, each with a barrier: 4 granules per thread

// A running maximum and sum of 2^(c (x - m)).  With hi = c m rounded, c x - hi is one multiply-add;
// the sum so formed is 2^d times the wanted one, d = c m - hi (one multiply-add too), and it is set right at the end.
// d is up to half of hi's last place: at most 1/2 below 2^24.  From there on, and where there is no maximum yet, the
// difference is taken first, which costs one more instruction a term: 2^d grows until it leaves binary32, from hi =
// 2^31 on (a mask of -1e10, or logits of 4 at a temperature of 1e-9).
template <typename W> struct Running {
    W m, s, hi;
    bool far;
};

__device__ __forceinline__ void refer(Running<float> &r, float m, float c) {
    r.m = m;
    r.hi = m * c;
    r.far = !(fabsf(r.hi) < 0x1p24f);
    if (r.far) r.hi = 0.0f;
}
__device__ __forceinline__ void refer(Running<double> &r, double m, double) { r.m = m, r.far = true, r.hi = 0; }

// The factor that the terms of r are too large by.
__device__ __forceinline__ float excess(const Running<float> &r, float c) {
    return r.far ? 1.0f : fast_exp2(fmaf(r.m, c, -r.hi));
}
__device__ __forceinline__ double excess(const Running<double> &, double) { return 1.0; }

template <typename W> __device__ __forceinline__ W term(const Running<W> &r, W x, W c) {
    return r.far ? fast_exp2((x - r.m) * c) : fast_exp2(fma(x, c, -r.hi));
}

// A new, larger maximum: the sum is taken relative to it.
template <typename W> __device__ __forceinline__ void raise(Running<W> &r, W m, W c) {
    const Running<W> old = r;
    refer(r, m, c);
    if (old.s != W(0))
        r.s = old.far || r.far ? old.s / excess(old, c) * excess(r, c) * fast_exp2((old.m - m) * c)
                               : old.s * fast_exp2(old.hi - r.hi);
}

__device__ __forceinline__ void bulk_load(void *dst, const void *src, uint32_t bytes, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_addr(dst)),
        "l"(src), "r"(bytes), "r"(smem_addr(bar))
        : "memory");
}

// The joint maximum and sum of two shares (true sums, no excess).  A share without a finite logit has
// m = -infinity and s = 0; a NaN sum stays.
template <typename W> __device__ __forceinline__ void join(W &m, W &s, W m2, W s2, W c) {
    const W top = fmax(m, m2);
    s = (m == top || s == W(0) || isnan(s) ? s : s * fast_exp2((m - top) * c)) +
        (m2 == top || s2 == W(0) || isnan(s2) ? s2 : s2 * fast_exp2((m2 - top) * c));
    m = top;
}

template <typename T> __global__ void __launch_bounds__(kDistillThreads, 3) distill_slice_kernel(const DistillParams<T> p) {
    using W = WideOf<T>;
    constexpr int V = 16 / sizeof(T), WARPS = kDistillThreads / 32;
    in_stream_order();
    if (!chain_admits(p.guard)) return;  // the same answer in every CTA of the grid
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ uint64_t landed[kMostChunks];
    __shared__ W part_m[WARPS], part_s[WARPS], share[2];
    __shared__ double part_a[WARPS], part_sums[2][WARPS];
    __shared__ int part_flags[WARPS], repeated;
    uint32_t ranks;
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
    const uint32_t rank = cluster_rank();
    const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
    const uint64_t row = blockIdx.x / ranks;
    const T *z = p.logits + row * p.stride;
    // this CTA's elements [v0, v1) of the row, cut at the row's granules
    const uint32_t phase = (uint32_t)(reinterpret_cast<uintptr_t>(z) % 16 / sizeof(T));
    const int vocab = (int)p.vocab;
    const int v0 = max(0, (int)((int64_t)rank * p.slice) - (int)phase);
    const int v1 = (int)min((int64_t)vocab, (int64_t)(rank + 1) * p.slice - phase);
    const int lead = rank == 0 ? (int)phase : 0;  // elements of the first granule in front of v0
    const int count = max(0, v1 - v0), granules = (lead + count + V - 1) / V;
    const int whole0 = lead ? 1 : 0, whole1 = (lead + count) / V;  // granules [whole0, whole1) are not cut
    T *slice = reinterpret_cast<T *>(smem);  // element v at slice[lead + v - v0]
    double *prob = reinterpret_cast<double *>(smem + p.slice_bytes);
    int *place = reinterpret_cast<int *>(prob + p.k), *claimed = place + (p.k + 1) / 2 * 2;
    const int chunks = (granules * 16 + kChunk - 1) / kChunk;
    T *g = p.gradient ? p.gradient + row * p.gradient_stride : nullptr;
    const W weight = p.weights ? p.weights[row] : W(1), c = p.to_log2;
    const double t_inverse = p.t_inverse;

    // First of all the slice is sent for (whole granules by bulk copies), and the first 256 of the teacher's
    // entries, which are looked at while the slice is on its way.
    int64_t index = -1;
    W top_logit = 0;
    if (tid < p.k) index = p.indices[row * p.k + tid], top_logit = p.top[row * p.k + tid];
    if (tid == 0) {
        for (int i = 0; i < chunks; ++i) mbar_init(&landed[i], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        repeated = 0;
    }
    for (int j = tid; j < p.claims; j += kDistillThreads) claimed[j] = -1;
    if (tid < V) {  // the elements of cut granules
        const W absent = -INFINITY;
        if (lead) slice[tid] = tid < lead || tid - lead >= count ? Elem<T>::round(absent) : z[v0 + tid - lead];
        const int at = whole1 * V + tid;
        if (whole1 < granules && (whole1 > 0 || !lead))
            slice[at] = at - lead < count ? z[v0 + at - lead] : Elem<T>::round(absent);
    }
    __syncthreads();
    auto fill = [&](T *to, W value) {  // the slice's part of a row
        const T each = Elem<T>::round(value);
        alignas(16) T many[V];
#pragma unroll
        for (int e = 0; e < V; ++e) many[e] = each;
        const int odd = (int)((16 - reinterpret_cast<uintptr_t>(to + v0) % 16) % 16 / sizeof(T));
        const int head = min(count, odd), body = (count - head) / V;
        for (int i = tid; i < body; i += kDistillThreads)
            __stcs(reinterpret_cast<uint4 *>(to + v0 + head) + i, *reinterpret_cast<const uint4 *>(many));
        if (tid < head) to[v0 + tid] = each;
        if (tid < count - head - body * V) to[v0 + head + body * V + tid] = each;
    };
    auto nothing_to_learn = [&] {
        if (tid == 0 && rank == 0) {
            if (p.loss) p.loss[row] = W(0);
            if (p.stats_out) p.stats_out[2 * row] = W(0), p.stats_out[2 * row + 1] = W(1);
        }
        if (g) fill(g, W(0));
    };
    if (weight == W(0)) return nothing_to_learn();  // in every CTA of the cluster
    if (tid == 0)
        for (int i = 0; i < chunks; ++i) {
            const int a = max(whole0, i * (kChunk / 16)), b = min(whole1, (i + 1) * (kChunk / 16));
            if (b > a) {
                mbar_expect_tx(&landed[i], (uint32_t)(b - a) * 16);
                bulk_load(slice + a * V, z + v0 + (a * V - lead), (uint32_t)(b - a) * 16, &landed[i]);
            } else {
                mbar_arrive(&landed[i]);
            }
        }

    // the teacher's entries: t, -infinity for absent ones (t / T could be an infinity where t - max t is not).  (One copy of the code for all of
    // them: what is not in the instruction cache comes slowly while the memory is busy.)
    double a_max = -INFINITY;
    int flags = 0;  // 1: an entry is present, 2: one is bad
#pragma unroll 1
    for (int j = tid; j < p.k; j += kDistillThreads) {
        if (j >= kDistillThreads) index = p.indices[row * p.k + j], top_logit = p.top[row * p.k + j];
        const double t = (double)top_logit;
        bool there = index >= 0 && t != -INFINITY;
        if (there && (index >= vocab || !isfinite(t))) flags |= 2, there = false;
        if (there) flags |= 1;
        place[j] = there ? (int)index : -1;
        prob[j] = there ? t : -INFINITY;
        a_max = fmax(a_max, prob[j]);
    }
    if (p.k > 32 * warp) {
#pragma unroll
        for (int o = 16; o; o >>= 1) a_max = fmax(a_max, __shfl_xor_sync(~0u, a_max, o));
        flags = __reduce_or_sync(~0u, flags);
    }
    if (lane == 0) part_a[warp] = a_max, part_flags[warp] = flags;
    __syncthreads();
    a_max = part_a[0], flags = part_flags[0];
#pragma unroll
    for (int i = 1; i < WARPS; ++i) a_max = fmax(a_max, part_a[i]), flags |= part_flags[i];
    if (!flags) {  // in every CTA of the cluster
        nothing_to_learn();
        if (tid == 0)
            for (int i = 0; i < chunks; ++i) mbar_wait(&landed[i], 0);  // nothing is left in flight
        return;
    }

    // The sums over the entries, with a_j = (t_j - max t) / T and e_j = exp(a_j):
    //   mass = sum e_j, lean = sum e_j (a_j - (z_j - m) / T),
    // from which loss / (w T^2) = lean / mass + ln s - ln mass.  A table notes whether an index appears twice
    // (see the end).
    double mass = 0, lean = 0;
#pragma unroll 1
    for (int j = tid; j < p.k; j += kDistillThreads) {
        const int at = place[j];
        if (at < 0) continue;
        const double a = (prob[j] - a_max) * t_inverse, e = exp(a);
        mass += e;
        if (e > 0) lean += e * a;
        prob[j] = e;
        if (g) {
            unsigned probe = (unsigned)at * 2654435761u;
#pragma unroll 1
            for (;; ++probe) {  // at most half of the table is taken
                const int was = atomicCAS(&claimed[probe & (p.claims - 1)], -1, at);
                if (was == at) repeated = 1;
                if (was == -1 || was == at) break;
            }
        }
    }

    bool ok = true;
    W m, s, inverse;
    Running<W> run;
    if (p.stats_in) {
        m = p.stats_in[2 * row];
        s = p.stats_in[2 * row + 1];
    } else {
        refer(run, -INFINITY, c);
        run.s = W(0);
        alignas(16) T nothing[V];
        for (int e = 0; e < V; ++e) nothing[e] = Elem<T>::round(W(-INFINITY));
        const uint4 absent = *reinterpret_cast<const uint4 *>(nothing);
        for (int i = 0; i < chunks; ++i) {
            ok = ok && mbar_wait(&landed[i], 0);
            if (i * (kChunk / 16) + warp * 32 >= granules) break;  // the warp has no granule in this last chunk
            W x[4][V];
            W top = -INFINITY;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int at = i * (kChunk / 16) + q * kDistillThreads + tid;
                uint4 raw = absent;
                if (at < granules) raw = *reinterpret_cast<const uint4 *>(slice + at * V);
                unpack<T>(raw, x[q]);
                top = fmax(top, largest<T>(raw, x[q]));
            }
            if (top > run.m) raise(run, top, c);
            if (run.m == -INFINITY) {  // nothing but masked entries so far, or NaN
#pragma unroll
                for (int q = 0; q < 4; ++q)
#pragma unroll
                    for (int e = 0; e < V; ++e)
                        if (isnan(x[q][e])) run.s = x[q][e];
            } else if (run.far) {
#pragma unroll
                for (int q = 0; q < 4; ++q)
#pragma unroll
                    for (int e = 0; e < V; ++e) run.s += fast_exp2((x[q][e] - run.m) * c);
            } else {
                W sum[4] = {};
#pragma unroll
                for (int e = 0; e < V; ++e)
#pragma unroll
                    for (int q = 0; q < 4; ++q) sum[q] += fast_exp2(fma(x[q][e], c, -run.hi));
                run.s += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            }
        }
        m = run.m;
        s = run.s / excess(run, c);
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            const W m2 = __shfl_xor_sync(~0u, m, o), s2 = __shfl_xor_sync(~0u, s, o);
            join(m, s, m2, s2, c);
        }
        if (lane == 0) part_m[warp] = m, part_s[warp] = s;
    }
    // The first CTA's loss takes the logits that the teacher names, those of other CTAs' slices before any
    // CTA overwrites them in place: a thread's first one is kept in a register, further ones in the table's place.
    const bool losing = p.loss && rank == 0 && p.k > 32 * warp;
    auto named = [&](int j) {
        const int at = place[j];
        return at < 0 ? Elem<T>::round(W(0)) : at < v1 ? slice[lead + at - v0] : z[at];
    };
    T first_named = Elem<T>::round(W(0)), *further_named = reinterpret_cast<T *>(claimed) - kDistillThreads;
    if (losing && tid < p.k) first_named = named(tid);
    if (p.k > 32 * warp)
#pragma unroll
        for (int o = 16; o; o >>= 1) mass += __shfl_xor_sync(~0u, mass, o);
    if (lane == 0) part_sums[0][warp] = mass;

    if (!p.stats_in) {
        __syncthreads();
        if (losing)
#pragma unroll 1
            for (int j = tid + kDistillThreads; j < p.k; j += kDistillThreads) further_named[j] = named(j);
        // One warp joins the warps' shares, and the cluster's: always the same tree, so the same bits in
        // every CTA.
        auto joined = [&](int shares) {
#pragma unroll
            for (int o = 1; o < 8; o *= 2)
                if (o < shares) {
                    const W m2 = __shfl_xor_sync(~0u, m, o), s2 = __shfl_xor_sync(~0u, s, o);
                    // lower lanes' shares first on both sides
                    W ma = lane & o ? m2 : m, sa = lane & o ? s2 : s;
                    join(ma, sa, lane & o ? m : m2, lane & o ? s : s2, c);
                    m = ma, s = sa;
                }
        };
        static_assert(WARPS == 8, "as many warps as CTAs in the largest cluster");
        if (warp == 0) {
            m = part_m[lane % WARPS], s = part_s[lane % WARPS];
            joined(WARPS);
            if (lane == 0) share[0] = m, share[1] = s;
        }
        if (ranks > 1) {
            cluster_sync();
            if (warp == 0) {
                W m2, s2;
                cluster_read(m2, smem_addr(&share[0]), lane % ranks);
                cluster_read(s2, smem_addr(&share[1]), lane % ranks);
                m = m2, s = s2;
                joined((int)ranks);
                if (lane == 0) part_m[0] = m, part_s[0] = s;
            }
            // read; this CTA waits for the others' readings when it ends
            asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
        }
        __syncthreads();
        m = ranks > 1 ? part_m[0] : share[0], s = ranks > 1 ? part_s[0] : share[1];
    }
    auto over_warps = [&](const double (&part)[WARPS]) {  // behind a barrier
        double all = part[0];
#pragma unroll
        for (int i = 1; i < WARPS; ++i) all += part[i];
        return all;
    };
    const W up = p.upstream ? p.upstream[p.upstream_uniform ? 0 : row] : W(1);
    const bool invalid = (flags & 2) || !isfinite(m) || !isfinite(s) || !(s > W(0)) || !isfinite(weight) || (g && !isfinite(up));
    unsigned kind = invalid && tid == 0 ? (unsigned)PCU_B200_KIND_INVALID : 0u;
    if (rank == 0 && tid == 0 && p.stats_out) p.stats_out[2 * row] = m, p.stats_out[2 * row + 1] = s;
    // Each z_j - m by itself: of logits that share a large offset the differences count, and sum e_j z_j - m mass
    // would lose them (a row of -1e20 throughout had a loss of 1e4 for ln V - H(p)).
    if (losing) {
#pragma unroll 1
        for (int j = tid; j < p.k; j += kDistillThreads) {
            const double zj = (double)Elem<T>::load(j == tid ? first_named : further_named[j]);
            if (place[j] >= 0 && prob[j] > 0) lean -= prob[j] * ((zj - (double)m) * t_inverse);
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) lean += __shfl_xor_sync(~0u, lean, o);
    }
    if (lane == 0) part_sums[1][warp] = lean;
    if (g && invalid) {
        fill(g, W(NAN));
    } else if (g) {
        const W factor = up * weight * p.temperature;
        refer(run, m, c);
        inverse = W(1) / s / excess(run, c);
        const W scale = factor * inverse;
        // q is at most 1, so a result can only exceed its type where the factor does.  NaN and infinities
        // among the logits, which a backward call meets here first, stay in the sum `seen`.
        const bool check = !isfinite(Elem<T>::load(Elem<T>::round(factor)));
        W seen = 0;
        unsigned worst = 0;
        const bool aligned = (reinterpret_cast<uintptr_t>(g + v0) - lead * sizeof(T)) % 16 == 0;
        // plain: neither far nor check; first: no pass has read the slice yet
        auto sweep = [&](auto plain_, auto first_) {
            constexpr bool plain = decltype(plain_)::value, first = decltype(first_)::value;
            auto value = [&](W x) {
                const W e = plain ? fast_exp2(fma(x, c, -run.hi)) : term(run, x, c);
                if (first) seen += e;
                if (!plain && check) worst = max(worst, result_kind(Elem<T>::load(Elem<T>::round(scale * e))));
                return scale * e;
            };
            if (aligned) {
                for (int i = 0; i < chunks; ++i) {
                    if (first) ok = ok && mbar_wait(&landed[i], 0);
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const int at = i * (kChunk / 16) + q * kDistillThreads + tid;
                        if (at >= granules) break;
                        W x[V];
                        unpack<T>(*reinterpret_cast<const uint4 *>(slice + at * V), x);
#pragma unroll
                        for (int e = 0; e < V; ++e) x[e] = value(x[e]);
                        const uint4 packed = pack<T>(x);
                        T *to = g + v0 + (at * V - lead);
                        if (at >= whole0 && at < whole1) {
                            __stcs(reinterpret_cast<uint4 *>(to), packed);
                        } else {
#pragma unroll
                            for (int e = 0; e < V; ++e)
                                if (at * V + e >= lead && at * V + e - lead < count) to[e] = reinterpret_cast<const T *>(&packed)[e];
                        }
                    }
                }
            } else {  // the gradient's rows lie differently: element by element, adjacent lanes adjacent elements
                if (first)
                    for (int i = 0; i < chunks; ++i) ok = ok && mbar_wait(&landed[i], 0);
#pragma unroll 8
                for (int v = tid; v < count; v += kDistillThreads)
                    g[v0 + v] = Elem<T>::round(value(Elem<T>::load(slice[lead + v])));
            }
        };
        if (run.far || check) p.stats_in ? sweep(std::false_type{}, std::true_type{}) : sweep(std::false_type{}, std::false_type{});
        else p.stats_in ? sweep(std::true_type{}, std::true_type{}) : sweep(std::true_type{}, std::false_type{});
        if (!isfinite(seen) && !kind) kind = PCU_B200_KIND_INVALID;
        __syncthreads();  // before the entries' elements are written again
        mass = over_warps(part_sums[0]);
        for (int j = tid; j < p.k; j += kDistillThreads) {
            const int at = place[j];
            if (at < v0 || at >= v1) continue;
            double sum = prob[j];
            if (repeated) {  // the first entry of an index carries the sum of all of them
                bool first = true;
                for (int i = 0; i < j; ++i) first &= place[i] != at;
                if (!first) continue;
                for (int i = j + 1; i < p.k; ++i)
                    if (place[i] == at) sum += prob[i];
            }
            const W q = term(run, Elem<T>::load(slice[lead + at - v0]), c) * inverse;
            const T r = Elem<T>::round(factor * (q - (W)(sum / mass)));
            worst = max(worst, result_kind(Elem<T>::load(r)));
            g[at] = r;
        }
        if (worst && !kind) kind = worst;
    }
    if (p.loss && rank == 0) {
        __syncthreads();
        if (tid == 0) {
            mass = over_warps(part_sums[0]), lean = over_warps(part_sums[1]);
            const double t = (double)p.temperature;
            const W value = invalid ? W(NAN) : (W)((double)weight * t * t * (lean / mass + log((double)s) - log(mass)));
            p.loss[row] = value;
            if (const unsigned lost = result_kind(value)) record_fault(p.status, row, lost);
        }
    }
    if (!ok) record_fault(p.status, 0, kWatchdog);
    if (kind) record_fault(p.status, row, kind);
    // nothing is left in flight towards this CTA's shared memory, and the cluster has read it
    if (tid == 0)
        for (int i = 0; i < chunks; ++i) mbar_wait(&landed[i], 0);
    __syncwarp();
    if (!p.stats_in && ranks > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
}

// Rows go through shared memory where a cluster of 8 holds one.  The smallest cluster whose slices are
// at most 64 KB is taken (three such CTAs per SM overlap each other's phases); with fewer rows than
// fill the SMs twice, larger ones down to slices of 8 KB.
template <typename T>
static int launch_distill(DistillParams<T> p, uint64_t rows, cudaStream_t stream) {
    // the bytes that a row's granules span: 16 more where rows can start inside one
    const bool cut = reinterpret_cast<uintptr_t>(p.logits) % 16 || (rows > 1 && p.stride * sizeof(T) % 16);
    const uint64_t bytes = (p.vocab * sizeof(T) + 15) / 16 * 16 + (cut ? 16 : 0), sms = (uint64_t)pcu_host::sm_count();
    unsigned ranks = 1;
    while (ranks < 8 && bytes > ranks * 65536ull) ranks *= 2;
    while (ranks < 8 && rows * ranks < 2 * sms && bytes > ranks * 16384ull) ranks *= 2;
    const uint64_t slice_bytes = (bytes / 16 + ranks - 1) / ranks * 16;
    p.claims = 1;
    while (p.claims < 2 * p.k) p.claims *= 2;
    const uint64_t need = slice_bytes + (uint64_t)p.k * sizeof(double) + (uint64_t)((p.k + 1) / 2 * 2 + p.claims) * sizeof(int);
    if (slice_bytes > (uint64_t)kMostChunks * kChunk || need > 216 * 1024 || rows * ranks > 0x7fffffffull) {
        return pcu_host::launch_grid(distill_kernel<T>, (unsigned)rows, kDistillThreads, stream, p);
    }
    p.slice = (int)(slice_bytes / sizeof(T));
    p.slice_bytes = (uint32_t)slice_bytes;
    if (const int rc = pcu_host::allow_shared<distill_slice_kernel<T>>(216 * 1024)) return rc;
    return pcu_host::launch_cluster(distill_slice_kernel<T>, (unsigned)(rows * ranks), kDistillThreads, need, ranks, stream, p);
}

// The arguments that the three calls share; a call leaves out what it does not have.
struct DistillCall {
    int dtype;
    const void *logits;
    uint64_t rows, vocab, stride;
    const int64_t *indices;
    const void *top;
    uint64_t k;
    const void *weights;
    uint32_t temperature_bits;
    bool wants_loss, wants_gradient;
    void *loss, *stats_out;
    const void *stats_in, *upstream;
    int upstream_uniform;
    void *gradient;
    uint64_t gradient_stride;
    uint64_t *status;
    void *stream;
};

template <typename T> static int run_distill(const DistillCall &c, const ChainGuard &guard) {
    using W = WideOf<T>;
    DistillParams<T> p{};
    p.logits = (const T *)c.logits;
    p.vocab = c.vocab;
    p.stride = c.stride;
    p.indices = c.indices;
    p.top = (const W *)c.top;
    p.k = (int)c.k;
    p.weights = (const W *)c.weights;
    p.temperature = (W)pcu_host::rate_f32(c.temperature_bits);
    p.to_log2 = (W)(1.4426950408889634074 / (double)p.temperature);
    p.t_inverse = 1.0 / (double)p.temperature;
    p.loss = (W *)c.loss;
    p.stats_out = (W *)c.stats_out;
    p.stats_in = (const W *)c.stats_in;
    p.upstream = (const W *)c.upstream;
    p.upstream_uniform = c.upstream_uniform != 0;
    p.gradient = (T *)c.gradient;
    p.gradient_stride = c.gradient_stride;
    p.status = reinterpret_cast<unsigned long long *>(c.status);
    p.guard = guard;
    return launch_distill<T>(p, c.rows, pcu_host::as_stream(c.stream));
}

int distill(const DistillCall &c, const ChainGuard &guard) {
    if (!pcu_host::element_bytes(c.dtype) || !c.status) return PCU_B200_ERROR_INVALID_ARGUMENT;
    const float t = pcu_host::rate_f32(c.temperature_bits);
    if (!std::isnormal(t) || t < 0) return PCU_B200_ERROR_INVALID_ARGUMENT;
    if (c.rows == 0) return chain_decide_only(guard, pcu_host::as_stream(c.stream));
    if (c.vocab == 0 || c.stride < c.vocab || !c.logits) return PCU_B200_ERROR_INVALID_ARGUMENT;
    if (c.k && (!c.indices || !c.top)) return PCU_B200_ERROR_INVALID_ARGUMENT;
    if (c.wants_loss && !c.loss) return PCU_B200_ERROR_INVALID_ARGUMENT;
    if (c.wants_gradient && (!c.gradient || c.gradient_stride < c.vocab)) return PCU_B200_ERROR_INVALID_ARGUMENT;
    if (!c.wants_loss && !c.stats_in) return PCU_B200_ERROR_INVALID_ARGUMENT;
    const size_t bytes = pcu_host::element_bytes(c.dtype), wide = c.dtype == PCU_B200_F64 ? 8 : 4;
    for (const void *p : {c.logits, (const void *)c.gradient})
        if (!pcu_host::aligned(p, bytes)) return PCU_B200_ERROR_INVALID_ARGUMENT;
    for (const void *p : {c.top, c.weights, (const void *)c.loss, (const void *)c.stats_out, c.stats_in, c.upstream})
        if (!pcu_host::aligned(p, wide)) return PCU_B200_ERROR_INVALID_ARGUMENT;
    if (!pcu_host::aligned(c.indices, 8) || !pcu_host::aligned(c.status, 8)) return PCU_B200_ERROR_INVALID_ARGUMENT;
    // in place means the same rows: any other overlap would overwrite logits before they are read
    if (c.gradient == c.logits && c.wants_gradient && c.gradient_stride != c.stride) return PCU_B200_ERROR_INVALID_ARGUMENT;
    if (c.rows > 0x7fffffffull || c.vocab > 0x7fffffffull || c.k > PCU_B200_DISTILL_TOP_MAX ||
        c.stride > (1ull << 40) || c.gradient_stride > (1ull << 40))
        return PCU_B200_ERROR_SIZE_OVERFLOW;
    switch (c.dtype) {
    case PCU_B200_F32: return run_distill<float>(c, guard);
    case PCU_B200_F64: return run_distill<double>(c, guard);
    case PCU_B200_F16: return run_distill<__half>(c, guard);
    default: return run_distill<__nv_bfloat16>(c, guard);
    }
}

}  // namespace pcu

using pcu::ChainGuard;
using pcu::DistillCall;

static DistillCall loss_call(int dtype, const void *logits, uint64_t rows, uint64_t vocab, uint64_t logits_stride,
                             const int64_t *top_indices, const void *top_logits, uint64_t top_count,
                             const void *row_weights, uint32_t temperature_bits_f32, uint64_t *status, void *stream) {
    DistillCall c{};
    c.dtype = dtype;
    c.logits = logits;
    c.rows = rows;
    c.vocab = vocab;
    c.stride = logits_stride;
    c.indices = top_indices;
    c.top = top_logits;
    c.k = top_count;
    c.weights = row_weights;
    c.temperature_bits = temperature_bits_f32;
    c.status = status;
    c.stream = stream;
    return c;
}

#define PCU_DISTILL_INPUTS                                                                                          \
    int dtype, const void *logits, uint64_t rows, uint64_t vocab, uint64_t logits_stride,                           \
        const int64_t *top_indices, const void *top_logits, uint64_t top_count, const void *row_weights,            \
        uint32_t temperature_bits_f32
#define PCU_DISTILL_CALL(status)                                                                                    \
    loss_call(dtype, logits, rows, vocab, logits_stride, top_indices, top_logits, top_count, row_weights,           \
              temperature_bits_f32, status, stream)

namespace {

int forward(DistillCall c, void *loss, void *row_stats, const ChainGuard &guard) {
    c.wants_loss = true;
    c.loss = loss;
    c.stats_out = row_stats;
    if (c.rows && !row_stats) return PCU_B200_ERROR_INVALID_ARGUMENT;
    return pcu::distill(c, guard);
}

int backward(DistillCall c, const void *row_stats, const void *upstream, int upstream_uniform, void *gradient,
             uint64_t gradient_stride, const ChainGuard &guard) {
    c.wants_gradient = true;
    c.stats_in = row_stats;
    c.upstream = upstream;
    c.upstream_uniform = upstream_uniform;
    c.gradient = gradient;
    c.gradient_stride = gradient_stride;
    return pcu::distill(c, guard);
}

int step(DistillCall c, void *loss, void *row_stats, const void *upstream, int upstream_uniform, void *gradient,
         uint64_t gradient_stride, const ChainGuard &guard) {
    c.wants_loss = c.wants_gradient = true;
    c.loss = loss;
    c.stats_out = row_stats;
    c.upstream = upstream;
    c.upstream_uniform = upstream_uniform;
    c.gradient = gradient;
    c.gradient_stride = gradient_stride;
    return pcu::distill(c, guard);
}

}  // namespace

extern "C" int pcu_b200_distill_loss(PCU_DISTILL_INPUTS, void *loss, void *row_stats, uint64_t *status, void *stream) {
    return forward(PCU_DISTILL_CALL(status), loss, row_stats, ChainGuard{});
}

extern "C" int pcu_b200_distill_loss_backward(PCU_DISTILL_INPUTS, const void *row_stats, const void *upstream,
                                              int upstream_uniform, void *gradient, uint64_t gradient_stride,
                                              uint64_t *status, void *stream) {
    return backward(PCU_DISTILL_CALL(status), row_stats, upstream, upstream_uniform, gradient, gradient_stride,
                    ChainGuard{});
}

extern "C" int pcu_b200_distill_loss_step(PCU_DISTILL_INPUTS, void *loss, void *row_stats, const void *upstream,
                                          int upstream_uniform, void *gradient, uint64_t gradient_stride,
                                          uint64_t *status, void *stream) {
    return step(PCU_DISTILL_CALL(status), loss, row_stats, upstream, upstream_uniform, gradient, gradient_stride,
                ChainGuard{});
}

extern "C" int pcu_b200_guarded_distill_loss(PCU_DISTILL_INPUTS, void *loss, void *row_stats, uint64_t *chain_records,
                                             uint32_t chain_stage, void *stream) {
    if (!chain_records) return PCU_B200_ERROR_INVALID_ARGUMENT;
    return forward(PCU_DISTILL_CALL(chain_records + 2ull * chain_stage), loss, row_stats,
                   pcu_host::slab_guard(chain_records, chain_stage));
}

extern "C" int pcu_b200_guarded_distill_loss_backward(PCU_DISTILL_INPUTS, const void *row_stats, const void *upstream,
                                                      int upstream_uniform, void *gradient, uint64_t gradient_stride,
                                                      uint64_t *chain_records, uint32_t chain_stage, void *stream) {
    if (!chain_records) return PCU_B200_ERROR_INVALID_ARGUMENT;
    return backward(PCU_DISTILL_CALL(chain_records + 2ull * chain_stage), row_stats, upstream, upstream_uniform,
                    gradient, gradient_stride, pcu_host::slab_guard(chain_records, chain_stage));
}

extern "C" int pcu_b200_guarded_distill_loss_step(PCU_DISTILL_INPUTS, void *loss, void *row_stats, const void *upstream,
                                                  int upstream_uniform, void *gradient, uint64_t gradient_stride,
                                                  uint64_t *chain_records, uint32_t chain_stage, void *stream) {
    if (!chain_records) return PCU_B200_ERROR_INVALID_ARGUMENT;
    return step(PCU_DISTILL_CALL(chain_records + 2ull * chain_stage), loss, row_stats, upstream, upstream_uniform,
                gradient, gradient_stride, pcu_host::slab_guard(chain_records, chain_stage));
}
