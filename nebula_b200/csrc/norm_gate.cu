// Norms before and after a block, fused with its gate, its residual scale and the residual sum (no counterpart in the
// reference): per row
//   n = norm(x) * weight + bias          root mean square, or mean and variance, over the row or each of its groups
//   u = n * gate function(gate)
//   s = residual + scale * channel_scale * u
//   y = norm(s) * next_weight + next_bias   over the row: what the next block reads
// A row stays in registers from its loads to its stores, so every tensor crosses HBM once; sums are fp32.  The second norm reads s
// before it is rounded for storage.
#include <cuda_bf16.h>

#include "device_math.cuh"
#include "nb_internal.h"

namespace nb {

namespace {

struct NormParams {
    const void *x, *gate, *residual;
    void *sum, *y;
    const float *weight, *bias, *channel_scale, *next_weight, *next_bias;
    long long x_stride, gate_stride, residual_stride, sum_stride, y_stride;
    long long rows;
    int width, groups;          // of a row; groups > 1 only in the general kernel
    int fold;                   // > 0: a row here is one of `fold` groups of a row of the tensors
    int norm, next_norm, gate_mode;
    float eps, scale;
    int lanes;                  // threads of a row, a power of two
};

__device__ __forceinline__ float gate_value(float z, int mode) {
    if (mode == NB_GATE_LINEAR) return z;
    const float s = 1.0f / (1.0f + expf(-z));
    return mode == NB_GATE_SIGMOID ? s : z * s;
}

template <class T, int V> struct Raw;
template <> struct Raw<float, 4> { float4 r; __device__ float get(int i) const { return (&r.x)[i]; } };
template <> struct Raw<float, 1> { float r; __device__ float get(int) const { return r; } };
template <> struct Raw<__nv_bfloat16, 8> {
    uint4 r;
    __device__ float get(int i) const { const unsigned w = (&r.x)[i >> 1]; return __uint_as_float(i & 1 ? w & 0xffff0000u : w << 16); }
};
template <> struct Raw<__nv_bfloat16, 1> { __nv_bfloat16 r; __device__ float get(int) const { return __bfloat162float(r); } };
// a residual stream in fp32 beside blocks in bf16: eight values as two quads
template <> struct Raw<float, 8> { float4 r[2]; __device__ float get(int i) const { return (&r[i >> 2].x)[i & 3]; } };

template <class T, int V> __device__ __forceinline__ Raw<T, V> fetch(const void *p, long long at) { return *(const Raw<T, V> *)((const T *)p + at); }
template <class T, int V> __device__ __forceinline__ void put(void *p, long long at, const float *f) {
    if constexpr (sizeof(T) == 4) {
        if constexpr (V == 1) ((float *)p)[at] = f[0];
        else
#pragma unroll
            for (int i = 0; i < V; i += 4) *(float4 *)((float *)p + at + i) = make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]);
    } else if constexpr (V == 1) {
        ((__nv_bfloat16 *)p)[at] = __float2bfloat16_rn(f[0]);
    } else {
        uint4 r;
        __nv_bfloat162 *b = (__nv_bfloat162 *)&r;
#pragma unroll
        for (int i = 0; i < 4; i++) b[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
        *(uint4 *)((__nv_bfloat16 *)p + at) = r;
    }
}
template <int V> __device__ __forceinline__ void weights_at(const float *w, int at, float *f) {
    if constexpr (V == 1) f[0] = w[at];
    else
#pragma unroll
        for (int i = 0; i < V; i += 4) {
            const float4 v = *(const float4 *)(w + at + i);
            f[i] = v.x; f[i + 1] = v.y; f[i + 2] = v.z; f[i + 3] = v.w;
        }
}

// Sum over the threads of a row, the same for all of them.  Rows of up to a warp are segments of one; wider ones are a CTA of their
// own, whose warps' sums are added in order.
__device__ __forceinline__ float row_sum(float v, int lanes, float *red) {
    for (int o = min(lanes, 32) >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (lanes <= 32) return v;
    __syncthreads();            // the sums of the call before have been read
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = (threadIdx.x & 31) < (lanes >> 5) ? red[threadIdx.x & 31] : 0.0f;
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// The sum of f over each group of a row, `parts` being room for one value per vector of the row: every vector's sum goes
// there, and each group's are added by one warp in a fixed order.
template <int V, int NV, class F>
__device__ __forceinline__ void group_sums(const NormParams &p, float *parts, float *sums, F f) {
    const int vecs = p.width / V, per = vecs / p.groups, warps = (blockDim.x + 31) >> 5;
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NV; n++) {
        const int vec = n * p.lanes + threadIdx.x;
        if (vec < vecs) parts[vec] = f(n);
    }
    __syncthreads();
    for (int g = threadIdx.x >> 5; g < p.groups; g += warps) {
        float v = 0.0f;
        for (int i = threadIdx.x & 31; i < per; i += 32) v += parts[g * per + i];
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        if ((threadIdx.x & 31) == 0) sums[g] = v;
    }
    __syncthreads();
}

// T: type of x, gate and y.  R: type of residual and s.  V: values of one access.  NV: accesses of a thread.
// GROUPED: several groups a row (the first norm), for rows that a second norm joins again.
template <class T, class R, int V, int NV, bool GROUPED>
__global__ void __launch_bounds__(1024) norm_gate_kernel(NormParams p) {
    grid_begin();
    extern __shared__ float smem[];         // GROUPED: a value per vector of the row, then one per group
    __shared__ float red[32];
    const int lane = threadIdx.x & (p.lanes - 1);
    const long long row = (long long)blockIdx.x * (blockDim.x / p.lanes) + threadIdx.x / p.lanes;
    const bool live = row < p.rows;
    const long long r = p.fold ? row / p.fold : row;
    const int first = p.fold ? (int)(row % p.fold) * p.width : 0;
    float f[NV * V];
    Raw<T, V> gate[NV];
    Raw<R, V> res[NV];
#pragma unroll
    for (int n = 0; n < NV; n++) {
        const int c = (n * p.lanes + lane) * V;
        const bool in = live && c < p.width;
        Raw<T, V> x = {};
        gate[n] = {};
        res[n] = {};
        if (in) x = fetch<T, V>(p.x, r * p.x_stride + first + c);
        if (in && p.gate) gate[n] = fetch<T, V>(p.gate, r * p.gate_stride + first + c);
        if (in && p.residual) res[n] = fetch<R, V>(p.residual, r * p.residual_stride + first + c);
#pragma unroll
        for (int i = 0; i < V; i++) f[n * V + i] = x.get(i);
    }
    auto inside = [&](int n) { return (n * p.lanes + lane) * V < p.width; };
    auto normalise = [&](int mode) {
        float mean = 0.0f;
        if (mode == NB_NORM_LAYER) {
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < NV * V; i++) sum += f[i];
            mean = row_sum(sum, p.lanes, red) / p.width;
        }
        float power = 0.0f;
#pragma unroll
        for (int n = 0; n < NV; n++)
            if (inside(n))
#pragma unroll
                for (int i = 0; i < V; i++) {
                    f[n * V + i] -= mean;
                    power = fmaf(f[n * V + i], f[n * V + i], power);
                }
        const float by = 1.0f / sqrtf(row_sum(power, p.lanes, red) / p.width + p.eps);
#pragma unroll
        for (int i = 0; i < NV * V; i++) f[i] *= by;
    };
    if (p.norm != NB_NORM_NONE) {
        if constexpr (GROUPED) {
            float *parts = smem, *sums = smem + p.width / V;
            const int per = p.width / p.groups;
            if (p.norm == NB_NORM_LAYER) {
                group_sums<V, NV>(p, parts, sums, [&](int n) {
                    float s = 0.0f;
#pragma unroll
                    for (int i = 0; i < V; i++) s += f[n * V + i];
                    return s;
                });
#pragma unroll
                for (int n = 0; n < NV; n++)
                    if (inside(n)) {
                        const float mean = sums[(n * p.lanes + lane) * V / per] / per;
#pragma unroll
                        for (int i = 0; i < V; i++) f[n * V + i] -= mean;
                    }
            }
            group_sums<V, NV>(p, parts, sums, [&](int n) {
                float s = 0.0f;
#pragma unroll
                for (int i = 0; i < V; i++) s = fmaf(f[n * V + i], f[n * V + i], s);
                return s;
            });
#pragma unroll
            for (int n = 0; n < NV; n++)
                if (inside(n)) {
                    const float by = 1.0f / sqrtf(sums[(n * p.lanes + lane) * V / per] / per + p.eps);
#pragma unroll
                    for (int i = 0; i < V; i++) f[n * V + i] *= by;
                }
        } else {
            normalise(p.norm);
        }
    }
#pragma unroll
    for (int n = 0; n < NV; n++) {
        const int c = (n * p.lanes + lane) * V;
        if (live && c < p.width) {
            float w[V];
            if (p.weight) {
                weights_at<V>(p.weight, first + c, w);
#pragma unroll
                for (int i = 0; i < V; i++) f[n * V + i] *= w[i];
            }
            if (p.bias) {
                weights_at<V>(p.bias, first + c, w);
#pragma unroll
                for (int i = 0; i < V; i++) f[n * V + i] += w[i];
            }
            if (p.gate)
#pragma unroll
                for (int i = 0; i < V; i++) f[n * V + i] *= gate_value(gate[n].get(i), p.gate_mode);
            if (p.channel_scale) {
                weights_at<V>(p.channel_scale, first + c, w);
#pragma unroll
                for (int i = 0; i < V; i++) f[n * V + i] *= w[i];
            }
#pragma unroll
            for (int i = 0; i < V; i++) f[n * V + i] = fmaf(p.scale, f[n * V + i], p.residual ? res[n].get(i) : 0.0f);
            if (p.sum) put<R, V>(p.sum, r * p.sum_stride + first + c, f + n * V);
        }
    }
    if (p.next_norm == NB_NORM_NONE) return;
    normalise(p.next_norm);
#pragma unroll
    for (int n = 0; n < NV; n++) {
        const int c = (n * p.lanes + lane) * V;
        if (live && c < p.width) {
            float w[V];
            if (p.next_weight) {
                weights_at<V>(p.next_weight, first + c, w);
#pragma unroll
                for (int i = 0; i < V; i++) f[n * V + i] *= w[i];
            }
            if (p.next_bias) {
                weights_at<V>(p.next_bias, first + c, w);
#pragma unroll
                for (int i = 0; i < V; i++) f[n * V + i] += w[i];
            }
            put<T, V>(p.y, r * p.y_stride + first + c, f + n * V);
        }
    }
}

template <class T, class R, int V, int NV>
void launch_norm(nb_handle_s *h, const NormParams &p) {
    const int tpb = p.lanes > 32 ? p.lanes : 128;      // a row of more than a warp has a CTA of its own
    const dim3 grid((unsigned)((p.rows + tpb / p.lanes - 1) / (tpb / p.lanes)));
    const size_t smem = p.groups > 1 ? (size_t)(p.width / V + p.groups) * sizeof(float) : 0;
    NB_REQUIRE((p.rows + tpb / p.lanes - 1) / (tpb / p.lanes) < (1LL << 31), "norm: too many rows");
    if (p.groups > 1) {
        if (smem > 200 * 1024) throw Error(NB_ERR_UNSUPPORTED, "norm: too many groups in a row of this width");
        if (smem > 48 * 1024)
            NB_CHECK_CUDA(cudaFuncSetAttribute(norm_gate_kernel<T, R, V, NV, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        launch_overlapped(h, norm_gate_kernel<T, R, V, NV, true>, grid, tpb, smem, p);
    } else {
        launch_overlapped(h, norm_gate_kernel<T, R, V, NV, false>, grid, tpb, 0, p);
    }
    check_launch("norm_gate_kernel");
    count_launch(h);
}

constexpr int MAX_WIDTH = 32768;        // 1024 threads with 32 values each

// Threads and accesses of a row: as few threads as hold it with `most` accesses each, but rather more threads than a second
// access while the rows are fewer than the device's SMs.
template <class T, class R, int V>
void choose(nb_handle_s *h, NormParams p, int most) {
    const int vecs = (p.width + V - 1) / V;
    const int want = p.rows * 2 <= h->sm_count ? 1 : std::min(2, most);
    int lanes = p.groups > 1 ? 64 : 4;
    while (lanes < 1024 && lanes * want < vecs) lanes *= 2;
    p.lanes = lanes;
    const int nv = (vecs + lanes - 1) / lanes;
    if (nv <= 1) launch_norm<T, R, V, 1>(h, p);
    else if (nv <= 2) launch_norm<T, R, V, 2>(h, p);
    else if (nv <= 4) launch_norm<T, R, V, 4>(h, p);
    else if constexpr (V < 8) {
        if (nv <= 8) launch_norm<T, R, V, 8>(h, p);
        else if constexpr (V == 1) launch_norm<T, R, V, 32>(h, p);
    }
}

}  // namespace

void launch_norm_gate(nb_handle_s *h, const nb_norm_gate_desc_t &d, const nb_norm_gate_io_t &io) {
    NB_REQUIRE(d.rows >= 0 && d.width > 0 && d.groups > 0 && d.width % d.groups == 0, "norm: bad extent (groups divide the width)");
    if (d.width > MAX_WIDTH) throw Error(NB_ERR_UNSUPPORTED, "norm: rows of more than 32768 values");
    NB_REQUIRE(d.norm >= NB_NORM_NONE && d.norm <= NB_NORM_LAYER && d.next_norm >= NB_NORM_NONE && d.next_norm <= NB_NORM_LAYER, "norm: unknown norm");
    NB_REQUIRE(d.gate >= NB_GATE_NONE && d.gate <= NB_GATE_SILU, "norm: unknown gate function");
    NB_REQUIRE((d.dtype == NB_DTYPE_F32 || d.dtype == NB_DTYPE_BF16) && (d.residual_dtype == NB_DTYPE_F32 || d.residual_dtype == NB_DTYPE_BF16),
               "norm: unknown type");
    if (d.dtype == NB_DTYPE_F32 && d.residual_dtype == NB_DTYPE_BF16) throw Error(NB_ERR_UNSUPPORTED, "norm: a bf16 residual beside fp32 blocks");
    NB_REQUIRE(d.eps >= 0.0f, "norm: negative eps");
    if (d.rows == 0) return;
    NB_REQUIRE(io.x, "norm: null x");
    NB_REQUIRE((io.gate != nullptr) == (d.gate != NB_GATE_NONE), "norm: a gate and its function go together");
    NB_REQUIRE((io.y != nullptr) == (d.next_norm != NB_NORM_NONE), "norm: y and the second norm go together");
    NB_REQUIRE(io.sum || io.y, "norm: nothing to write");
    const size_t tb = d.dtype == NB_DTYPE_BF16 ? 2 : 4, rb = d.residual_dtype == NB_DTYPE_BF16 ? 2 : 4;
    NormParams p = {};
    size_t align = 0;           // addresses and strides in bytes, or-ed
    auto rows = [&](const void *ptr, long long stride, size_t bytes, const char *what) {
        const long long s = stride ? stride : d.width;
        if (!ptr) return s;
        NB_REQUIRE(s >= d.width || d.rows == 1, std::string("norm: row stride below the width: ") + what);
        NB_REQUIRE((uintptr_t)ptr % bytes == 0, std::string("norm: misaligned ") + what);
        check_extent(h, ptr, 0, ((d.rows - 1) * s + d.width) * (long long)bytes, what);
        align |= (uintptr_t)ptr | (size_t)(s * (long long)bytes);
        return s;
    };
    p.x_stride = rows(io.x, d.x_stride, tb, "x");
    p.gate_stride = rows(io.gate, d.gate_stride, tb, "gate");
    p.residual_stride = rows(io.residual, d.residual_stride, rb, "residual");
    p.sum_stride = rows(io.sum, d.sum_stride, rb, "sum");
    p.y_stride = rows(io.y, d.y_stride, tb, "y");
    for (const float *w : {io.weight, io.bias, io.channel_scale, io.next_weight, io.next_bias}) {
        if (!w) continue;
        NB_REQUIRE((uintptr_t)w % 4 == 0, "norm: misaligned weights");
        check_extent(h, w, 0, (long long)d.width * 4, "norm weights");
        align |= (uintptr_t)w;
    }
    p.x = io.x; p.gate = io.gate; p.residual = io.residual; p.sum = io.sum; p.y = io.y;
    p.weight = io.weight; p.bias = io.bias; p.channel_scale = io.channel_scale; p.next_weight = io.next_weight; p.next_bias = io.next_bias;
    p.rows = d.rows; p.width = d.width; p.groups = d.norm == NB_NORM_NONE ? 1 : d.groups;
    p.norm = d.norm; p.next_norm = d.next_norm; p.gate_mode = d.gate; p.eps = d.eps; p.scale = d.scale;
    if (p.groups > 1 && p.next_norm == NB_NORM_NONE) {      // nothing joins the groups again: each is a row of its own
        p.fold = p.groups;
        p.rows *= p.groups;
        p.width /= p.groups;
        p.groups = 1;
    }
    // whole accesses of 16 bytes: every row, group and vector of weights starts on such a boundary and is made of whole ones
    const int v = d.dtype == NB_DTYPE_BF16 ? 8 : 4;
    const bool whole = align % 16 == 0 && p.width % v == 0 && p.width / p.groups % v == 0;
    if (d.dtype == NB_DTYPE_F32) {
        if (whole) choose<float, float, 4>(h, p, 8);
        else choose<float, float, 1>(h, p, 32);
    } else if (d.residual_dtype == NB_DTYPE_BF16) {
        if (whole) choose<__nv_bfloat16, __nv_bfloat16, 8>(h, p, 4);
        else choose<__nv_bfloat16, __nv_bfloat16, 1>(h, p, 32);
    } else {
        if (whole) choose<__nv_bfloat16, float, 8>(h, p, 4);
        else choose<__nv_bfloat16, float, 1>(h, p, 32);
    }
}

}  // namespace nb
