// Bias of the channels-first linear layer: y[b, c, :] += bias[c], and its gradient
// gbias[c] = sum over samples and positions of gy[b, c, :]; and the same bias fused with the
// erf-form GELU that follows the first projection of the network's MLP: a = gelu(h + bias) in
// one pass over h, and gh = ga * gelu'(h + bias) with the bias gradient in one pass over (ga, h).
//
// The 1x1 projection itself is a library GEMM; what the library adds around it, a broadcast add
// that is not vectorised and a reduction with one block per output, is slow at the small per-GPU
// batches of a batch-sharded training step.  Both are plain HBM-bound passes here: every
// (sample, channel) slab is split over as many CTAs as fill the GPU, 16-byte accesses, sums in a
// fixed order (no atomics).
#include <cstdarg>
#include <cstdio>

#include "ndc_b200.h"
#include "ndc_common.cuh"
#include "ndc_gelu.cuh"
#include "ndc_slab.cuh"

namespace {

using namespace ndc::gelu;
using namespace ndc::slab;

thread_local char g_bias_err[256] = "";

int bias_fail(int status, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_bias_err, sizeof(g_bias_err), fmt, ap);
    va_end(ap);
    return status;
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kNT) bias_add_kernel(T* __restrict__ y, long long sp, int channels,
                                                       int nsplit, const float* __restrict__ bias) {
    const long long slab = blockIdx.x / nsplit;
    const int part = blockIdx.x % nsplit;
    T* ys = y + slab * sp;
    const float b = bias[slab % channels];
    long long begin, end;
    part_range(sp, nsplit, part, Vec16<T>::N, begin, end);
    constexpr int N = Vec16<T>::N;
    if (VEC) {
        for (long long i = begin + (long long)threadIdx.x * N; i < end; i += (long long)kNT * N) {
            float v[N];
            Vec16<T>::unpack(*reinterpret_cast<const typename Vec16<T>::raw*>(ys + i), v);
#pragma unroll
            for (int j = 0; j < N; ++j) v[j] += b;
            *reinterpret_cast<typename Vec16<T>::raw*>(ys + i) = Vec16<T>::pack(v);
        }
    } else {
        for (long long i = begin + threadIdx.x; i < end; i += kNT)
            ys[i] = ndc::from_f32<T>(ndc::to_f32(ys[i]) + b);
    }
}

// y = v + bias rounded once: v of whole rows of `count` values, y's rows `pitch` apart.
template <bool VEC>
__global__ void __launch_bounds__(kNT) bias_round_kernel(const float* __restrict__ v, __nv_bfloat16* __restrict__ y, long long count, long long pitch,
                                                         int channels, int nsplit, const float* __restrict__ bias) {
    typedef Vec16<__nv_bfloat16> V;
    const long long slab = blockIdx.x / nsplit;
    const int part = blockIdx.x % nsplit;
    const float* vs = v + slab * count;
    __nv_bfloat16* ys = y + slab * pitch;
    const float b = bias[slab % channels];
    long long begin, end;
    part_range(count, nsplit, part, V::N, begin, end);
    if (VEC) {
        for (long long i = begin + (long long)threadIdx.x * V::N; i < end; i += (long long)kNT * V::N) {
            const float4 lo = *reinterpret_cast<const float4*>(vs + i), hi = *reinterpret_cast<const float4*>(vs + i + 4);
            const float f[8] = {lo.x + b, lo.y + b, lo.z + b, lo.w + b, hi.x + b, hi.y + b, hi.z + b, hi.w + b};
            *reinterpret_cast<V::raw*>(ys + i) = V::pack(f);
        }
    } else {
        for (long long i = begin + threadIdx.x; i < end; i += kNT) ys[i] = __float2bfloat16_rn(vs[i] + b);
    }
}

// partial[slab * nsplit + part] = sum of the part
template <typename T, bool VEC>
__global__ void __launch_bounds__(kNT) bias_grad_partial_kernel(const T* __restrict__ gy, long long sp,
                                                                int nsplit, float* __restrict__ partial) {
    __shared__ float scratch[2 * kNT / 32];
    const long long slab = blockIdx.x / nsplit;
    const int part = blockIdx.x % nsplit;
    const T* gs = gy + slab * sp;
    long long begin, end;
    part_range(sp, nsplit, part, Vec16<T>::N, begin, end);
    constexpr int N = Vec16<T>::N;
    float s1 = 0.0f, s2 = 0.0f;     // two interleaved sums: shorter dependency chains
    if (VEC) {
        for (long long i = begin + (long long)threadIdx.x * N; i < end; i += (long long)kNT * N) {
            float v[N];
            Vec16<T>::unpack(__ldg(reinterpret_cast<const typename Vec16<T>::raw*>(gs + i)), v);
#pragma unroll
            for (int j = 0; j < N; j += 2) { s1 += v[j]; s2 += v[j + 1]; }
        }
    } else {
        for (long long i = begin + threadIdx.x; i < end; i += kNT) s1 += ndc::to_f32(gs[i]);
    }
    cta_sum2(s1, s2, scratch);
    if (threadIdx.x == 0) partial[slab * nsplit + part] = s1 + s2;
}

__global__ void bias_grad_final_kernel(const float* __restrict__ partial, int batch, int channels, int nsplit,
                                       float* __restrict__ gbias) {
    const int c = blockIdx.x * blockDim.x + threadIdx.x;
    if (c >= channels) return;
    float s = 0.0f;
    for (int b = 0; b < batch; ++b)
        for (int i = 0; i < nsplit; ++i) s += partial[((long long)b * channels + c) * nsplit + i];
    gbias[c] = s;
}

constexpr int kGeluUnroll = 4;     // 16-byte loads in flight per thread and tensor

template <typename T, bool VEC>
__global__ void __launch_bounds__(kNT) bias_gelu_fwd_kernel(const T* __restrict__ h, T* __restrict__ out,
                                                            long long sp, int channels, int nsplit,
                                                            const float* __restrict__ bias) {
    const long long slab = blockIdx.x / nsplit;
    const int part = blockIdx.x % nsplit;
    const T* hs = h + slab * sp;
    T* os = out + slab * sp;
    const float b = bias ? bias[slab % channels] : 0.0f;
    long long begin, end;
    part_range(sp, nsplit, part, Vec16<T>::N, begin, end);
    constexpr int N = Vec16<T>::N;
    if (VEC) {
        // kGeluUnroll independent 16-byte loads per thread are issued before the first erf: the
        // arithmetic of one vector is long enough to leave the memory pipe idle otherwise
        typedef typename Vec16<T>::raw Raw;
        const long long step = (long long)kNT * N;
        const f2 b2 = f2_dup(b);
        long long i = begin + (long long)threadIdx.x * N;
        for (; i + (kGeluUnroll - 1) * step < end; i += kGeluUnroll * step) {
            Raw r[kGeluUnroll];
#pragma unroll
            for (int u = 0; u < kGeluUnroll; ++u) r[u] = __ldg(reinterpret_cast<const Raw*>(hs + i + u * step));
#pragma unroll
            for (int u = 0; u < kGeluUnroll; ++u) {
                float v[N];
                Vec16<T>::unpack(r[u], v);
#pragma unroll
                for (int j = 0; j < N; j += 2)
                    f2_unpack(gelu2(f2_add(f2_pack(v[j], v[j + 1]), b2)), v[j], v[j + 1]);
                *reinterpret_cast<Raw*>(os + i + u * step) = Vec16<T>::pack(v);
            }
        }
        for (; i < end; i += step) {
            float v[N];
            Vec16<T>::unpack(__ldg(reinterpret_cast<const Raw*>(hs + i)), v);
#pragma unroll
            for (int j = 0; j < N; j += 2)
                f2_unpack(gelu2(f2_add(f2_pack(v[j], v[j + 1]), b2)), v[j], v[j + 1]);
            *reinterpret_cast<Raw*>(os + i) = Vec16<T>::pack(v);
        }
    } else {
        for (long long i = begin + threadIdx.x; i < end; i += kNT)
            os[i] = ndc::from_f32<T>(gelu_f(ndc::to_f32(hs[i]) + b));
    }
}

// gh = ga * gelu'(h + bias), rounded to the storage type; partial[slab * nsplit + part] = the
// sum of the rounded values of the part (what a separate pass over gh would add up)
template <typename T, bool VEC>
__global__ void __launch_bounds__(kNT) bias_gelu_bwd_kernel(const T* __restrict__ ga, const T* __restrict__ h,
                                                            T* __restrict__ gh, long long sp, int channels,
                                                            int nsplit, const float* __restrict__ bias,
                                                            float* __restrict__ partial) {
    __shared__ float scratch[2 * kNT / 32];
    const long long slab = blockIdx.x / nsplit;
    const int part = blockIdx.x % nsplit;
    const T* gs = ga + slab * sp;
    const T* hs = h + slab * sp;
    T* os = gh + slab * sp;
    const float b = bias ? bias[slab % channels] : 0.0f;
    long long begin, end;
    part_range(sp, nsplit, part, Vec16<T>::N, begin, end);
    constexpr int N = Vec16<T>::N;
    float s1 = 0.0f, s2 = 0.0f;
    if (VEC) {
        typedef typename Vec16<T>::raw Raw;
        const long long step = (long long)kNT * N;
        const f2 b2 = f2_dup(b);
        auto one = [&](const Raw& rg, const Raw& rh, long long at) {
            float g[N], v[N];
            Vec16<T>::unpack(rg, g);
            Vec16<T>::unpack(rh, v);
#pragma unroll
            for (int j = 0; j < N; j += 2)
                f2_unpack(f2_mul(f2_pack(g[j], g[j + 1]), gelu_grad2(f2_add(f2_pack(v[j], v[j + 1]), b2))),
                          g[j], g[j + 1]);
            const Raw r = Vec16<T>::pack(g);
            *reinterpret_cast<Raw*>(os + at) = r;
            Vec16<T>::unpack(r, g);
#pragma unroll
            for (int j = 0; j < N; j += 2) { s1 += g[j]; s2 += g[j + 1]; }
        };
        long long i = begin + (long long)threadIdx.x * N;
        for (; i + (kGeluUnroll - 1) * step < end; i += kGeluUnroll * step) {
            Raw rg[kGeluUnroll], rh[kGeluUnroll];
#pragma unroll
            for (int u = 0; u < kGeluUnroll; ++u) {
                rg[u] = __ldg(reinterpret_cast<const Raw*>(gs + i + u * step));
                rh[u] = __ldg(reinterpret_cast<const Raw*>(hs + i + u * step));
            }
#pragma unroll
            for (int u = 0; u < kGeluUnroll; ++u) one(rg[u], rh[u], i + u * step);
        }
        for (; i < end; i += step)
            one(__ldg(reinterpret_cast<const Raw*>(gs + i)), __ldg(reinterpret_cast<const Raw*>(hs + i)), i);
    } else {
        for (long long i = begin + threadIdx.x; i < end; i += kNT) {
            const T r = ndc::from_f32<T>(ndc::to_f32(gs[i]) * gelu_grad_f(ndc::to_f32(hs[i]) + b));
            os[i] = r;
            s1 += ndc::to_f32(r);
        }
    }
    if (partial) {
        cta_sum2(s1, s2, scratch);
        if (threadIdx.x == 0) partial[slab * nsplit + part] = s1 + s2;
    }
}

int check(int32_t batch, int32_t channels, int64_t spatial, int32_t dtype) {
    if (batch <= 0 || channels <= 0 || spatial <= 0)
        return bias_fail(NDC_ERR_INVALID, "bias: batch, channels and spatial size must be positive");
    if (dtype != NDC_F32 && dtype != NDC_BF16)
        return bias_fail(NDC_ERR_INVALID, "bias: dtype must be NDC_F32 or NDC_BF16");
    if ((long long)batch * channels * kMaxSplit > 0x7fffffffLL)
        return bias_fail(NDC_ERR_UNSUPPORTED, "bias: batch * channels is too large");
    return NDC_OK;
}

}  // namespace

extern "C" {

const char* ndc_bias_last_error(void) { return g_bias_err; }

size_t ndc_bias_grad_workspace_bytes(int32_t batch, int32_t channels) {
    if (batch <= 0 || channels <= 0) return 0;
    return (size_t)batch * channels * kMaxSplit * sizeof(float);
}

int ndc_bias_add(int32_t batch, int32_t channels, int64_t spatial, int32_t dtype, void* y,
                 const float* bias, void* stream) {
    if (!y || !bias) return bias_fail(NDC_ERR_INVALID, "bias add: y and bias must not be NULL");
    int st = check(batch, channels, spatial, dtype);
    if (st != NDC_OK) return st;
    const long long slabs = (long long)batch * channels;
    const int nsplit = choose_split(slabs, spatial);
    const bool vec = spatial % (dtype == NDC_BF16 ? 8 : 4) == 0 && ((uintptr_t)y % 16) == 0;
    const unsigned grid = (unsigned)(slabs * nsplit);
    cudaStream_t s = (cudaStream_t)stream;
    if (dtype == NDC_F32) {
        if (vec) bias_add_kernel<float, true><<<grid, kNT, 0, s>>>((float*)y, spatial, channels, nsplit, bias);
        else bias_add_kernel<float, false><<<grid, kNT, 0, s>>>((float*)y, spatial, channels, nsplit, bias);
    } else {
        typedef __nv_bfloat16 bf16;
        if (vec) bias_add_kernel<bf16, true><<<grid, kNT, 0, s>>>((bf16*)y, spatial, channels, nsplit, bias);
        else bias_add_kernel<bf16, false><<<grid, kNT, 0, s>>>((bf16*)y, spatial, channels, nsplit, bias);
    }
    ndc::launched();
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return bias_fail(NDC_ERR_CUDA, "bias add: %s", cudaGetErrorString(e));
    return NDC_OK;
}

int ndc_bias_round(int32_t batch, int32_t channels, int64_t count, const float* v, const float* bias, void* y, int64_t pitch, void* stream) {
    if (!v || !bias || !y) return bias_fail(NDC_ERR_INVALID, "bias round: v, bias and y must not be NULL");
    const int st = check(batch, channels, count, NDC_BF16);
    if (st != NDC_OK) return st;
    if (pitch < count) return bias_fail(NDC_ERR_INVALID, "bias round: rows overlap");
    if (((uintptr_t)v | (uintptr_t)bias) % 4 || (uintptr_t)y % 2) return bias_fail(NDC_ERR_ALIGNMENT, "bias round: a tensor does not lie on its elements' size");
    const long long slabs = (long long)batch * channels;
    const int nsplit = choose_split(slabs, count);
    const bool vec = count % 8 == 0 && pitch % 8 == 0 && ((uintptr_t)v | (uintptr_t)y) % 16 == 0;
    const unsigned grid = (unsigned)(slabs * nsplit);
    cudaStream_t s = (cudaStream_t)stream;
    typedef __nv_bfloat16 bf16;
    if (vec) bias_round_kernel<true><<<grid, kNT, 0, s>>>(v, (bf16*)y, count, pitch, channels, nsplit, bias);
    else bias_round_kernel<false><<<grid, kNT, 0, s>>>(v, (bf16*)y, count, pitch, channels, nsplit, bias);
    ndc::launched();
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return bias_fail(NDC_ERR_CUDA, "bias round: %s", cudaGetErrorString(e));
    return NDC_OK;
}

int ndc_bias_grad(int32_t batch, int32_t channels, int64_t spatial, int32_t dtype, const void* gy,
                  float* gbias, void* workspace, size_t workspace_bytes, void* stream) {
    if (!gy || !gbias) return bias_fail(NDC_ERR_INVALID, "bias gradient: gy and gbias must not be NULL");
    int st = check(batch, channels, spatial, dtype);
    if (st != NDC_OK) return st;
    if (!workspace || workspace_bytes < ndc_bias_grad_workspace_bytes(batch, channels))
        return bias_fail(NDC_ERR_WORKSPACE, "bias gradient: workspace of %zu bytes needed",
                         ndc_bias_grad_workspace_bytes(batch, channels));
    const long long slabs = (long long)batch * channels;
    const int nsplit = choose_split(slabs, spatial);
    const bool vec = spatial % (dtype == NDC_BF16 ? 8 : 4) == 0 && ((uintptr_t)gy % 16) == 0;
    const unsigned grid = (unsigned)(slabs * nsplit);
    cudaStream_t s = (cudaStream_t)stream;
    float* partial = (float*)workspace;
    if (dtype == NDC_F32) {
        if (vec) bias_grad_partial_kernel<float, true><<<grid, kNT, 0, s>>>((const float*)gy, spatial, nsplit, partial);
        else bias_grad_partial_kernel<float, false><<<grid, kNT, 0, s>>>((const float*)gy, spatial, nsplit, partial);
    } else {
        typedef __nv_bfloat16 bf16;
        if (vec) bias_grad_partial_kernel<bf16, true><<<grid, kNT, 0, s>>>((const bf16*)gy, spatial, nsplit, partial);
        else bias_grad_partial_kernel<bf16, false><<<grid, kNT, 0, s>>>((const bf16*)gy, spatial, nsplit, partial);
    }
    bias_grad_final_kernel<<<(channels + 127) / 128, 128, 0, s>>>(partial, batch, channels, nsplit, gbias);
    ndc::launched(2);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return bias_fail(NDC_ERR_CUDA, "bias gradient: %s", cudaGetErrorString(e));
    return NDC_OK;
}

int ndc_bias_gelu_fwd(int32_t batch, int32_t channels, int64_t spatial, int32_t dtype, const void* h,
                      const float* bias, void* out, void* stream) {
    if (!h || !out) return bias_fail(NDC_ERR_INVALID, "bias gelu: h and out must not be NULL");
    int st = check(batch, channels, spatial, dtype);
    if (st != NDC_OK) return st;
    const long long slabs = (long long)batch * channels;
    const int nsplit = choose_split(slabs, spatial);
    const bool vec = spatial % (dtype == NDC_BF16 ? 8 : 4) == 0 && ((uintptr_t)h % 16) == 0 &&
                     ((uintptr_t)out % 16) == 0;
    const unsigned grid = (unsigned)(slabs * nsplit);
    cudaStream_t s = (cudaStream_t)stream;
    if (dtype == NDC_F32) {
        if (vec) bias_gelu_fwd_kernel<float, true><<<grid, kNT, 0, s>>>((const float*)h, (float*)out, spatial, channels, nsplit, bias);
        else bias_gelu_fwd_kernel<float, false><<<grid, kNT, 0, s>>>((const float*)h, (float*)out, spatial, channels, nsplit, bias);
    } else {
        typedef __nv_bfloat16 bf16;
        if (vec) bias_gelu_fwd_kernel<bf16, true><<<grid, kNT, 0, s>>>((const bf16*)h, (bf16*)out, spatial, channels, nsplit, bias);
        else bias_gelu_fwd_kernel<bf16, false><<<grid, kNT, 0, s>>>((const bf16*)h, (bf16*)out, spatial, channels, nsplit, bias);
    }
    ndc::launched();
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return bias_fail(NDC_ERR_CUDA, "bias gelu: %s", cudaGetErrorString(e));
    return NDC_OK;
}

int ndc_bias_gelu_bwd(int32_t batch, int32_t channels, int64_t spatial, int32_t dtype, const void* ga,
                      const void* h, const float* bias, void* gh, float* gbias, void* workspace,
                      size_t workspace_bytes, void* stream) {
    if (!ga || !h || !gh) return bias_fail(NDC_ERR_INVALID, "bias gelu gradient: ga, h and gh must not be NULL");
    int st = check(batch, channels, spatial, dtype);
    if (st != NDC_OK) return st;
    if (gbias && (!workspace || workspace_bytes < ndc_bias_grad_workspace_bytes(batch, channels)))
        return bias_fail(NDC_ERR_WORKSPACE, "bias gelu gradient: workspace of %zu bytes needed",
                         ndc_bias_grad_workspace_bytes(batch, channels));
    const long long slabs = (long long)batch * channels;
    const int nsplit = choose_split(slabs, spatial);
    const bool vec = spatial % (dtype == NDC_BF16 ? 8 : 4) == 0 && ((uintptr_t)ga % 16) == 0 &&
                     ((uintptr_t)h % 16) == 0 && ((uintptr_t)gh % 16) == 0;
    const unsigned grid = (unsigned)(slabs * nsplit);
    cudaStream_t s = (cudaStream_t)stream;
    float* partial = gbias ? (float*)workspace : nullptr;
    if (dtype == NDC_F32) {
        if (vec) bias_gelu_bwd_kernel<float, true><<<grid, kNT, 0, s>>>((const float*)ga, (const float*)h, (float*)gh, spatial, channels, nsplit, bias, partial);
        else bias_gelu_bwd_kernel<float, false><<<grid, kNT, 0, s>>>((const float*)ga, (const float*)h, (float*)gh, spatial, channels, nsplit, bias, partial);
    } else {
        typedef __nv_bfloat16 bf16;
        if (vec) bias_gelu_bwd_kernel<bf16, true><<<grid, kNT, 0, s>>>((const bf16*)ga, (const bf16*)h, (bf16*)gh, spatial, channels, nsplit, bias, partial);
        else bias_gelu_bwd_kernel<bf16, false><<<grid, kNT, 0, s>>>((const bf16*)ga, (const bf16*)h, (bf16*)gh, spatial, channels, nsplit, bias, partial);
    }
    ndc::launched();
    if (gbias) {
        bias_grad_final_kernel<<<(channels + 127) / 128, 128, 0, s>>>(partial, batch, channels, nsplit, gbias);
        ndc::launched();
    }
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return bias_fail(NDC_ERR_CUDA, "bias gelu gradient: %s", cudaGetErrorString(e));
    return NDC_OK;
}

}  // extern "C"
