// group_norm.cu -- group norm with an activation, channels last, forward and backward.
//
// x[n][s][c], group g = c / D, D = channels / groups, m = positions * D elements per (n, g):
//   mean = sum x / m, var = sum (x - mean)^2 / m, r = 1 / sqrt(var + eps), h = (x - mean) r,
//   z = h w + b, y = act(z);
// backward: dz = dy act'(z), db = sum dz, dw = sum dz h (over n and s),
//   c1 = sum_g dz w / m, c2 = sum_g dz w h / m, dx = r (dz w - c1 - h c2).
#include "learn.cuh"
#include "provider.h"

namespace pcu {

constexpr int kNormThreads = 256;

// A channels-last tensor: element (n, s, c) at n * batch + s * row + c.
template <typename T> struct Maps {
    T *base;
    uint64_t batch, row;
    __device__ __forceinline__ T *at(uint64_t n, uint64_t s, uint64_t c) const { return base + n * batch + s * row + c; }
};

template <typename T> struct NormParams {
    using W = WideOf<T>;
    Maps<const T> x, dy;
    Maps<T> out;  // y, or dx
    const W *weight, *bias;
    W *stats_out;
    const W *stats;
    W *sums;  // workspace: (c1, c2) for each (n, g)
    W *dweight, *dbias;
    uint64_t batch, positions, channels, groups, width;
    W eps;
    unsigned long long *status;
    ChainGuard guard;
};

template <int ACT, typename W> __device__ __forceinline__ W activate(W z) {
    if (ACT == PCU_B200_ACTIVATION_RELU) return z < W(0) ? W(0) : z;  // NaN stays
    if (ACT == PCU_B200_ACTIVATION_SILU) return z / (W(1) + exp(-z));
    if (ACT == PCU_B200_ACTIVATION_GELU) return z * W(0.5) * erfc(z * W(-0.70710678118654752440));
    return z;
}

template <int ACT, typename W> __device__ __forceinline__ W slope(W z) {
    if (ACT == PCU_B200_ACTIVATION_RELU) return z > W(0) ? W(1) : W(0);
    if (ACT == PCU_B200_ACTIVATION_SILU) {
        const W q = W(1) / (W(1) + exp(-z));
        return q * (W(1) + z * (W(1) - q));
    }
    if (ACT == PCU_B200_ACTIVATION_GELU)
        return W(0.5) * erfc(z * W(-0.70710678118654752440)) + z * exp(W(-0.5) * z * z) * W(0.39894228040143267794);
    return W(1);
}

// act'(z) at z = h w + b, h = (x - mean) r.  ReLU's slope is a step, so a z within its own rounding
// error of 0 (h and the product are each off by a few 2^-24) is decided in binary64.
template <int ACT, typename W>
__device__ __forceinline__ W slope_at(W x, W mean, W r, W h, W w, W b) {
    const W z = h * w + b;
    if (ACT == PCU_B200_ACTIVATION_RELU && sizeof(W) == 4 && fabs(z) <= (fabs(h * w) + fabs(b)) * W(0x1p-20))
        return ((double)x - (double)mean) * (double)r * (double)w + (double)b > 0.0 ? W(1) : W(0);
    return slope<ACT>(z);
}

template <typename V> __device__ __forceinline__ V norm_block_sum(V v, V *scratch) {
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    __syncthreads();
    if (threadIdx.x % 32 == 0) scratch[threadIdx.x / 32] = v;
    __syncthreads();
    v = scratch[0];
    for (int i = 1; i < kNormThreads / 32; ++i) v += scratch[i];
    return v;
}

// One CTA per (n, g): the group's statistics.
template <typename T> __global__ void __launch_bounds__(kNormThreads) norm_stats_kernel(const NormParams<T> p) {
    using W = WideOf<T>;
    if (!chain_admits(p.guard)) return;
    __shared__ W scratch[kNormThreads / 32];
    const uint64_t n = blockIdx.x / p.groups, g = blockIdx.x % p.groups, m = p.positions * p.width;
    W sum = 0, square = 0;
    for (uint64_t i = threadIdx.x; i < m; i += kNormThreads)
        sum += Elem<T>::load(*p.x.at(n, i / p.width, g * p.width + i % p.width));
    const W mean = m ? norm_block_sum(sum, scratch) / (W)m : W(0);
    for (uint64_t i = threadIdx.x; i < m; i += kNormThreads) {
        const W d = Elem<T>::load(*p.x.at(n, i / p.width, g * p.width + i % p.width)) - mean;
        square += d * d;
    }
    const W var = m ? norm_block_sum(square, scratch) / (W)m : W(0);
    if (threadIdx.x == 0) {
        p.stats_out[2 * blockIdx.x] = mean;
        // a variance that is not finite has no reciprocal root to scale by: NaN, not 0
        p.stats_out[2 * blockIdx.x + 1] = isfinite(var) ? W(1) / sqrt(var + p.eps) : W(NAN);
    }
}

template <typename T, int ACT>
__global__ void __launch_bounds__(kNormThreads) norm_apply_kernel(const NormParams<T> p) {
    using W = WideOf<T>;
    if (!chain_admits(p.guard)) return;
    const uint64_t total = p.batch * p.positions * p.channels;
    for (uint64_t i = blockIdx.x * (uint64_t)kNormThreads + threadIdx.x; i < total;
         i += (uint64_t)gridDim.x * kNormThreads) {
        const uint64_t c = i % p.channels, s = i / p.channels % p.positions, n = i / p.channels / p.positions;
        const W *st = p.stats + 2 * (n * p.groups + c / p.width);
        const W h = (Elem<T>::load(*p.x.at(n, s, c)) - st[0]) * st[1];
        const W z = h * (p.weight ? p.weight[c] : W(1)) + (p.bias ? p.bias[c] : W(0));
        const T y = Elem<T>::round(activate<ACT>(z));
        *p.out.at(n, s, c) = y;
        if (const unsigned kind = result_kind(Elem<T>::load(y))) record_fault(p.status, i, kind);
    }
}

// One CTA per (n, g): c1 and c2.
template <typename T, int ACT>
__global__ void __launch_bounds__(kNormThreads) norm_sums_kernel(const NormParams<T> p) {
    using W = WideOf<T>;
    if (!chain_admits(p.guard)) return;
    __shared__ W scratch[kNormThreads / 32];
    const uint64_t n = blockIdx.x / p.groups, g = blockIdx.x % p.groups, m = p.positions * p.width;
    const W mean = p.stats[2 * blockIdx.x], r = p.stats[2 * blockIdx.x + 1];
    W c1 = 0, c2 = 0;
    for (uint64_t i = threadIdx.x; i < m; i += kNormThreads) {
        const uint64_t s = i / p.width, c = g * p.width + i % p.width;
        const W w = p.weight ? p.weight[c] : W(1), b = p.bias ? p.bias[c] : W(0);
        const W x = Elem<T>::load(*p.x.at(n, s, c)), h = (x - mean) * r;
        const W k = Elem<T>::load(*p.dy.at(n, s, c)) * slope_at<ACT>(x, mean, r, h, w, b) * w;
        c1 += k;
        c2 += k * h;
    }
    c1 = norm_block_sum(c1, scratch);
    c2 = norm_block_sum(c2, scratch);
    if (threadIdx.x == 0) p.sums[2 * blockIdx.x] = c1 / (W)m, p.sums[2 * blockIdx.x + 1] = c2 / (W)m;
}

// One CTA per channel: the parameters' gradients.
template <typename T, int ACT>
__global__ void __launch_bounds__(kNormThreads) norm_parameters_kernel(const NormParams<T> p) {
    using W = WideOf<T>;
    if (!chain_admits(p.guard)) return;
    __shared__ W scratch[kNormThreads / 32];
    const uint64_t c = blockIdx.x, rows = p.batch * p.positions;
    const W w = p.weight ? p.weight[c] : W(1), b = p.bias ? p.bias[c] : W(0);
    W dw = 0, db = 0;
    for (uint64_t i = threadIdx.x; i < rows; i += kNormThreads) {
        const uint64_t n = i / p.positions, s = i % p.positions;
        const W *st = p.stats + 2 * (n * p.groups + c / p.width);
        const W x = Elem<T>::load(*p.x.at(n, s, c)), h = (x - st[0]) * st[1];
        const W dz = Elem<T>::load(*p.dy.at(n, s, c)) * slope_at<ACT>(x, st[0], st[1], h, w, b);
        dw += dz * h;
        db += dz;
    }
    dw = norm_block_sum(dw, scratch);
    db = norm_block_sum(db, scratch);
    if (threadIdx.x != 0) return;
    const uint64_t first = rows * p.channels + c;
    if (p.dweight) {
        p.dweight[c] = dw;
        if (const unsigned kind = result_kind(dw)) record_fault(p.status, first, kind);
    }
    if (p.dbias) {
        p.dbias[c] = db;
        if (const unsigned kind = result_kind(db)) record_fault(p.status, first + p.channels, kind);
    }
}

template <typename T, int ACT>
__global__ void __launch_bounds__(kNormThreads) norm_gradient_kernel(const NormParams<T> p) {
    using W = WideOf<T>;
    if (!chain_admits(p.guard)) return;
    const uint64_t total = p.batch * p.positions * p.channels;
    for (uint64_t i = blockIdx.x * (uint64_t)kNormThreads + threadIdx.x; i < total;
         i += (uint64_t)gridDim.x * kNormThreads) {
        const uint64_t c = i % p.channels, s = i / p.channels % p.positions, n = i / p.channels / p.positions;
        const uint64_t at = 2 * (n * p.groups + c / p.width);
        const W mean = p.stats[at], r = p.stats[at + 1];
        const W w = p.weight ? p.weight[c] : W(1), b = p.bias ? p.bias[c] : W(0);
        const W x = Elem<T>::load(*p.x.at(n, s, c)), h = (x - mean) * r;
        const W k = Elem<T>::load(*p.dy.at(n, s, c)) * slope_at<ACT>(x, mean, r, h, w, b) * w;
        const T dx = Elem<T>::round(r * (k - p.sums[at] - h * p.sums[at + 1]));
        *p.out.at(n, s, c) = dx;
        if (const unsigned kind = result_kind(Elem<T>::load(dx))) record_fault(p.status, i, kind);
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

// 0 for what the calls refuse
size_t workspace_size(int dtype, uint64_t batch, uint64_t positions, uint64_t channels, uint64_t groups, bool backward) {
    if (!pcu_host::element_bytes(dtype) || groups == 0 || channels % groups != 0 ||
        !shape_fits(batch, positions, channels, groups))
        return 0;
    if (!backward) return 0;
    return (size_t)(2 * batch * groups * (dtype == PCU_B200_F64 ? 8 : 4));
}

template <typename T, int ACT> int run_norm(const NormCall &c, NormParams<T> p, cudaStream_t stream) {
    const uint64_t total = c.batch * c.positions * c.channels;
    const uint64_t want = (total + kNormThreads - 1) / kNormThreads, cap = (uint64_t)pcu_host::sm_count() * 8;
    const unsigned blocks = (unsigned)(want < cap ? (want ? want : 1) : cap);
    const unsigned groups = (unsigned)(c.batch * c.groups);
    int rc = PCU_B200_OK;
    if (!c.backward) {
        norm_stats_kernel<T><<<groups, kNormThreads, 0, stream>>>(p);
        if ((rc = pcu_host::launch_status())) return rc;
        p.guard = chain_follow(p.guard);
        norm_apply_kernel<T, ACT><<<blocks, kNormThreads, 0, stream>>>(p);
        return pcu_host::launch_status();
    }
    if (total) {
        norm_sums_kernel<T, ACT><<<groups, kNormThreads, 0, stream>>>(p);
        if ((rc = pcu_host::launch_status())) return rc;
        p.guard = chain_follow(p.guard);
    }
    if (p.dweight || p.dbias) {  // before the gradient, which may overwrite input or upstream
        norm_parameters_kernel<T, ACT><<<(unsigned)c.channels, kNormThreads, 0, stream>>>(p);
        if ((rc = pcu_host::launch_status())) return rc;
        p.guard = chain_follow(p.guard);
    }
    if (total) norm_gradient_kernel<T, ACT><<<blocks, kNormThreads, 0, stream>>>(p);
    return pcu_host::launch_status();
}

template <typename T> int typed_norm(const NormCall &c, const ChainGuard &guard) {
    using W = WideOf<T>;
    NormParams<T> p{};
    p.x = {(const T *)c.input, c.input_batch_stride, c.input_stride};
    p.dy = {(const T *)c.upstream, c.upstream_batch_stride, c.upstream_stride};
    p.out = {(T *)c.out, c.out_batch_stride, c.out_stride};
    p.weight = (const W *)c.weight;
    p.bias = (const W *)c.bias;
    p.stats_out = (W *)c.stats_out;
    p.stats = c.backward ? (const W *)c.stats_in : (const W *)c.stats_out;
    p.sums = (W *)c.workspace;
    p.dweight = (W *)c.dweight;
    p.dbias = (W *)c.dbias;
    p.batch = c.batch;
    p.positions = c.positions;
    p.channels = c.channels;
    p.groups = c.groups;
    p.width = c.channels / c.groups;
    p.eps = (W)pcu_host::rate_f32(c.eps_bits);
    p.status = reinterpret_cast<unsigned long long *>(c.status);
    p.guard = guard;
    cudaStream_t stream = pcu_host::as_stream(c.stream);
    switch (c.activation) {
    case PCU_B200_ACTIVATION_RELU: return run_norm<T, PCU_B200_ACTIVATION_RELU>(c, p, stream);
    case PCU_B200_ACTIVATION_SILU: return run_norm<T, PCU_B200_ACTIVATION_SILU>(c, p, stream);
    case PCU_B200_ACTIVATION_GELU: return run_norm<T, PCU_B200_ACTIVATION_GELU>(c, p, stream);
    default: return run_norm<T, PCU_B200_ACTIVATION_NONE>(c, p, stream);
    }
}

// Rows of `channels` elements: a batch's rows lie within its stride, so no two rows overlap.
bool good_maps(const void *base, uint64_t batch, uint64_t positions, uint64_t channels, uint64_t batch_stride,
               uint64_t stride) {
    if (!base) return false;
    if (positions > 1 && stride < channels) return false;
    const uint64_t reach = (positions - 1) * stride + channels;
    return batch <= 1 || batch_stride >= reach || (positions == 1 && batch_stride >= channels);
}

int norm(const NormCall &c, const ChainGuard &guard) {
    if (!pcu_host::element_bytes(c.dtype) || c.activation < 0 || c.activation > PCU_B200_ACTIVATION_GELU || !c.status)
        return PCU_B200_ERROR_INVALID_ARGUMENT;
    if (c.groups == 0 || c.channels % c.groups != 0) return PCU_B200_ERROR_INVALID_ARGUMENT;
    const float eps = pcu_host::rate_f32(c.eps_bits);
    if (!std::isfinite(eps) || std::signbit(eps)) return PCU_B200_ERROR_INVALID_ARGUMENT;
    if (!shape_fits(c.batch, c.positions, c.channels, c.groups) || c.input_batch_stride > kMost || c.input_stride > kMost || c.out_batch_stride > kMost || c.out_stride > kMost ||
        (c.backward && (c.upstream_batch_stride > kMost || c.upstream_stride > kMost)) ||
        !pcu_host::multiply_fits(c.input_stride, c.positions, kMost) ||
        !pcu_host::multiply_fits(c.out_stride, c.positions, kMost) ||
        (c.backward && !pcu_host::multiply_fits(c.upstream_stride, c.positions, kMost)))
        return PCU_B200_ERROR_SIZE_OVERFLOW;
    if (c.channels == 0 || (!c.backward && c.batch == 0) ||
        (c.backward && (c.batch == 0 || c.positions == 0) && !c.dweight && !c.dbias))
        return chain_decide_only(guard, pcu_host::as_stream(c.stream));
    if (!c.backward && !c.stats_out) return PCU_B200_ERROR_INVALID_ARGUMENT;
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
