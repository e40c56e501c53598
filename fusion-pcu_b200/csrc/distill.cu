// distill.cu -- distillation loss against a teacher's top logits, and its gradient.
//
// Row i has the student's logits z[0..V), the teacher's entries (idx_j, t_j), j < k, a weight w
// and an upstream gradient u.  With temperature T
//   q = softmax(z / T) over the vocabulary, p = softmax(t / T) over the row's present entries,
//   loss = w T^2 sum_j p_j (ln p_j - ln q[idx_j]),   d loss u / d z_v = u w T (q_v - sum_{idx_j = v} p_j).
// The row statistics are m = max z and s = sum exp((z - m) / T): q_v = exp((z_v - m) / T) / s keeps
// the relative precision of binary32, which a single log-sum-exp of magnitude 50 would not.
#include "learn.cuh"
#include "provider.h"

namespace pcu {

constexpr int kDistillThreads = 256;

template <typename T> struct DistillParams {
    using W = WideOf<T>;
    const T *logits;
    uint64_t vocab, stride;
    const int64_t *indices;
    const W *top;
    int k;
    const W *weights;
    W temperature, to_log2;  // T and log2(e) / T
    W *loss;                 // null: gradient only
    W *stats_out;            // may be null
    const W *stats_in;       // gradient only
    const W *upstream;       // null: 1
    int upstream_uniform;
    T *gradient;             // null: loss only
    uint64_t gradient_stride;
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

// One CTA per row.
template <typename T> __global__ void __launch_bounds__(kDistillThreads) distill_kernel(const DistillParams<T> p) {
    using W = WideOf<T>;
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
        prob[j] = there ? t / (double)p.temperature : -INFINITY;
        a_max = fmax(a_max, prob[j]);
    }
    a_max = block_max(a_max, scratch_d);
    bad = __syncthreads_or(bad);
    const bool skip = weight == W(0) || (a_max == -INFINITY && !bad);
    if (skip) {  // nothing to learn from: the row is not read
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
        if (place[j] >= 0) mass += exp(prob[j] - a_max);
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
        const double pj = exp(prob[j] - a_max) / mass;
        if (pj > 0)
            terms += pj * ((prob[j] - a_max - ln_mass) - ((zj - (double)m) / (double)p.temperature - log((double)s)));
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

template <typename T>
static int launch_distill(const DistillParams<T> &p, uint64_t rows, cudaStream_t stream) {
    distill_kernel<T><<<(unsigned)rows, kDistillThreads, 0, stream>>>(p);
    return pcu_host::launch_status();
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
