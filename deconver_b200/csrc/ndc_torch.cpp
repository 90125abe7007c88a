// The host path in native code: one autograd node for the whole `Deconv` layer (parameters ->
// float32, 1x1 projection, multiplicative updates), and one each for its neighbours in a block
// (1x1 projection with bias, bias + GELU, instance norm), on the C ABI of libndc_b200.so and cuBLAS.
//
// What bounds the layer at the deep stages and on single images is not the GPU: at 512 channels
// x 8^3 a forward and backward are 0.16 ms of kernels, and issuing them from Python through
// separate autograd nodes took 0.60 ms.  One node, one pass over the parameters in each
// direction, and no intermediate tensor that the update kernels do not read.  The neighbours the same:
// see the figures at their section.
#include <ATen/Context.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/ops/convolution_backward.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/relu.h>
#include <c10/cuda/CUDAGuard.h>
#include <cublas_v2.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <algorithm>
#include <mutex>
#include <tuple>
#include <vector>

#include "ndc_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

int dtype_code(const Tensor& t) { return t.scalar_type() == at::kBFloat16 ? NDC_BF16 : NDC_F32; }
bool kernel_dtype(const Tensor& t) { return t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16; }
// The tensor's memory.  A tensor may have none though it has elements (FakeTensor and other wrappers): library
// calls would read at address zero.
void* ptr(const Tensor& t) {
    if (!t.defined()) return nullptr;
    void* p = t.data_ptr();
    TORCH_CHECK(p || !t.numel(), "deconver_b200: a tensor of ", t.sizes(), " has no memory; the kernels need one that does");
    return p;
}
float* fptr(const Tensor& t) { return static_cast<float*>(ptr(t)); }
void* stream() { return at::cuda::getCurrentCUDAStream().stream(); }

void check(int status, const char* message) {
    TORCH_CHECK(status == NDC_OK, "ndc_b200 status ", status, ": ", message);
}

// The nodes have no forward-mode derivative.  Their own `apply` says so, but calls without reverse-mode
// gradients do not go through it, and would drop the tangents.
void refuse_tangents(std::initializer_list<const Tensor*> tensors) {
    for (const Tensor* t : tensors)
        TORCH_CHECK(!t->defined() || !t->_fw_grad(0).defined(), "deconver_b200: forward-mode differentiation is not implemented");
}

// ---- optional CUDA-event timing of ndc_fwd / ndc_bwd on the stream they are issued on ----------
struct Timing {
    std::mutex mu;
    bool enabled = false;
    std::vector<std::pair<cudaEvent_t, cudaEvent_t>> spans[2];   // forward, backward
} g_timing;

struct Span {
    cudaEvent_t start = nullptr, stop = nullptr;
    int kind;
    explicit Span(int k) : kind(k) {
        if (!g_timing.enabled) return;
        C10_CUDA_CHECK(cudaEventCreate(&start));
        C10_CUDA_CHECK(cudaEventCreate(&stop));
        C10_CUDA_CHECK(cudaEventRecord(start, (cudaStream_t)stream()));
    }
    ~Span() {
        if (!start) return;
        (void)cudaEventRecord(stop, (cudaStream_t)stream());
        std::lock_guard<std::mutex> lock(g_timing.mu);
        g_timing.spans[kind].emplace_back(start, stop);
    }
};

void timing_enable() {
    std::lock_guard<std::mutex> lock(g_timing.mu);
    for (auto& v : g_timing.spans) {
        for (auto& s : v) { (void)cudaEventDestroy(s.first); (void)cudaEventDestroy(s.second); }
        v.clear();
    }
    g_timing.enabled = true;
}

// Stops collecting; the caller has synchronised.  {forward ms, backward ms}
std::vector<std::vector<float>> timing_collect() {
    std::lock_guard<std::mutex> lock(g_timing.mu);
    g_timing.enabled = false;
    std::vector<std::vector<float>> out(2);
    for (int k = 0; k < 2; ++k) {
        for (auto& s : g_timing.spans[k]) {
            float ms = 0.0f;
            C10_CUDA_CHECK(cudaEventElapsedTime(&ms, s.first, s.second));
            out[k].push_back(ms);
            (void)cudaEventDestroy(s.first);
            (void)cudaEventDestroy(s.second);
        }
        g_timing.spans[k].clear();
    }
    return out;
}

// ---- 1x1 projections -------------------------------------------------------------------------
// The precision the framework gives convolutions of float32 tensors: TF32 unless switched off.
bool conv_tf32() { return at::globalContext().allowTF32CuDNN(at::Float32Op::CONV); }

// y[b] = op(w) x[b] (+ y[b] if `accumulate`) for a (Co, Ci) matrix `w`, op = transpose if
// `transpose`, and contiguous (B, channels, N) tensors: one strided batched library GEMM with the
// matrix repeated by a zero batch stride; no tensor is converted or copied.
void channel_gemm(const Tensor& w, bool transpose, const Tensor& x, Tensor& y, int64_t batch, int64_t n,
                  bool accumulate) {
    const int64_t co = w.size(0), ci = w.size(1);
    const int64_t out = transpose ? ci : co, in = transpose ? co : ci;
    if (!batch || !n || !out || !in) return;
    const bool bf16 = x.scalar_type() == at::kBFloat16;
    const bool tf32 = !bf16 && conv_tf32();
    const float one = 1.0f, beta = accumulate ? 1.0f : 0.0f;
    const cudaDataType_t type = bf16 ? CUDA_R_16BF : CUDA_R_32F;
    const cublasComputeType_t compute = tf32 ? CUBLAS_COMPUTE_32F_FAST_TF32 : CUBLAS_COMPUTE_32F;
    at::NoTF32Guard plain;   // the handle's own mode; `compute` says what this product uses
    cublasHandle_t handle = at::cuda::getCurrentCUDABlasHandle();
    // column-major view: (n x out) = (n x in) * (in x out)
    const cublasStatus_t st = cublasGemmStridedBatchedEx(
        handle, CUBLAS_OP_N, transpose ? CUBLAS_OP_T : CUBLAS_OP_N, (int)n, (int)out, (int)in, &one, ptr(x),
        type, (int)n, (long long)(in * n), ptr(w), type, (int)ci, 0LL, &beta, ptr(y), type, (int)n,
        (long long)(out * n), (int)batch, compute, CUBLAS_GEMM_DEFAULT);
    TORCH_CHECK(st == CUBLAS_STATUS_SUCCESS, "deconver_b200: projection GEMM failed (cuBLAS status ", (int)st, ")");
}

// The weight gradient of a 1x1 projection is a product of two wide matrices along their positions, and no
// one way is the fastest over the channels, batches and positions that occur:
//   Kernel       ndc_proj_wgrad: any row length; its MMAs' rate and tiles of 128 x 64 bound it for many channels
//   Product      one library product per sample, where samples and tiles of 128 x 128 fill the GPU
//   Slices       a sample's positions in 32 or 16 slices (more were slower: 2 x (256 + 64) x 262144 takes 136 us
//                with 32, 157 with 74), one batched library product per sample
//   Convolution  the library's convolution backward, for rows that are not whole vectors and many channels
// (Slices and Product are views of the tensors as they lie, float32 partial products, summed by ndc_proj_sum.)
enum WgradRoute { kKernel = 0, kProduct = 1, kSlices = 2, kConvolution = 3 };
struct WgradPlan { WgradRoute route; int64_t slices; };

// Whole vectors: the least expected time, microseconds, of the first three, by constants fitted to 1481
// float32 and 1317 bfloat16 shapes (16 to 2048 channels, 1 to 16 samples of 343 to 262144 positions).  On 400
// other shapes of either type the choice takes 42 and 51 ms together, the library's convolution 88 and
// 94, fixed limits on channels and batches (before) 55 and 57; by more than a tenth the convolution is
// faster on 39 and 7 (before: 135 and 76), but it is up to 50 times slower on others, which cannot be foreseen.
// Others (672 shapes): below the limit the kernel takes 0.05 - 0.9 times the library's convolution on the
// average of a class of widths and batches, above it 1.0 - 3.5; a single sample is a plain product for the
// library (1.3 - 3.8 from 20000 on).
// `exact` (float32 without TF32): the kernel throughout.  On 350 shapes it takes 0.42 times the library's
// convolution, and is off by 2.8e-7 of the result against 64 bits where the convolution is by 5.5e-7, slices by 7.2e-7
// and one product per sample, a single chain along its positions, by 1.4e-6 (1e-5 at most).
WgradPlan plan_weight_grad(int64_t batch, int64_t co, int64_t ci, int64_t n, bool bf16, bool exact, int sms) {
    if (exact) return {kKernel, 1};
    if (n % (bf16 ? 8 : 4)) {
        const int64_t limit = batch == 1 ? 20000 : batch <= 8 ? 200000 : bf16 ? 100000 : 30000;
        return {co * ci >= limit ? kConvolution : kKernel, 1};
    }
    const auto tiles = [](int64_t v, int64_t t) { return (v + t - 1) / t; };
    const double e = bf16 ? 2 : 4, bytes = (double)(co + ci) * n * e;                       // of a sample
    const int64_t square = tiles(co, 128) * tiles(ci, 128);
    // the library's products: CTAs of 128 x 128 outputs, each one chain along its positions
    const double rate = bf16 ? 1180.0 : n % 8 ? 455.0 : 525.0;                              // positions per us
    const double product = 14.0 + std::max((double)tiles(batch * square, sms) * n / rate, batch * bytes / 3.9e6);
    const int64_t slices = std::min<int64_t>(square < 4 ? 32 : 16, n / 1024);
    const double sliced = slices < 2 ? product + 1.0
                                     : 9.0 + (n % (8 * slices) ? 8.0 : 0.0) +
                                           batch * (5.5 + std::max(bytes / 5.0e6, 2.0 * co * ci * n / (bf16 ? 600e6 : 370e6)));
    // ndc_proj_wgrad: see plan_wgrad there
    const int64_t t = tiles(co, 128) * tiles(ci, 64), parts = std::max<int64_t>(1, std::min(tiles(4 * sms, t * batch), tiles(n, 512)));
    const double flops = 2.0 * batch * n * t * 128 * 64, read = ((double)co * tiles(ci, 64) + (double)ci * tiles(co, 128)) * batch * n * e;
    const double kernel = 7.3 + std::max(flops / (bf16 ? 272e6 : 134e6) / std::min(1.0, t * batch * parts / (2.0 * sms)), read / (bf16 ? 5.7e6 : 4.1e6)) +
                          batch * parts * co * ci * 8 / (bf16 ? 1.8e6 : 1.4e6);
    if (kernel <= product && kernel <= sliced) return {kKernel, 1};
    return product <= sliced ? WgradPlan{kProduct, 1} : WgradPlan{kSlices, slices};
}

Tensor weight_grad(const Tensor& gy, const Tensor& x, const Tensor& w, int64_t batch, int64_t n) {
    Tensor gw = at::empty(w.sizes(), w.options());
    const int64_t co = w.size(0), ci = w.size(1);
    if (!batch || !n || !co || !ci) return gw.zero_();
    const bool bf16 = gy.scalar_type() == at::kBFloat16;
    const WgradPlan plan = plan_weight_grad(batch, co, ci, n, bf16, !bf16 && !conv_tf32(), at::cuda::getCurrentDeviceProperties()->multiProcessorCount);
    if (plan.route == kConvolution)
        return std::get<1>(at::convolution_backward(gy.view({batch, co, n}), x.view({batch, ci, n}), w.view({co, ci, 1}), at::nullopt, {1}, {0},
                                                    {1}, false, {0}, 1, {false, true, false})).view(w.sizes());
    if (plan.route == kKernel) {
        const size_t bytes = ndc_proj_wgrad_workspace_bytes((int)batch, (int)co, (int)ci, n);
        Tensor ws = at::empty({(int64_t)bytes}, w.options().dtype(at::kByte));
        check(ndc_proj_wgrad((int)batch, (int)co, (int)ci, n, dtype_code(gy), conv_tf32() ? 1 : 0, ptr(gy), ptr(x),
                             ptr(gw), ptr(ws), bytes, stream()), ndc_proj_last_error());
        return gw;
    }
    // slices of whole vectors, and what they leave
    const int64_t slices = plan.slices, length = slices > 1 ? n / slices / 8 * 8 : n, rest = n - slices * length;
    Tensor partial = at::empty({batch * slices, co, ci}, w.options().dtype(at::kFloat));
    const cudaDataType_t type = bf16 ? CUDA_R_16BF : CUDA_R_32F;
    const cublasComputeType_t compute = bf16 ? CUBLAS_COMPUTE_32F : CUBLAS_COMPUTE_32F_FAST_TF32;
    at::NoTF32Guard plain;
    cublasHandle_t handle = at::cuda::getCurrentCUDABlasHandle();
    // `count` products along `k` positions, the first from position `at` of sample b on, the others
    // further on in it (`length` apart) or in the samples after it
    auto products = [&](int64_t b, int64_t at, int64_t k, bool samples, int64_t count, float beta) {
        const float one = 1.0f;
        const size_t e = bf16 ? 2 : 4;
        const int64_t sx = samples ? ci * n : length, sy = samples ? co * n : length, out_step = samples ? slices : 1;
        const cublasStatus_t st = cublasGemmStridedBatchedEx(
            handle, CUBLAS_OP_T, CUBLAS_OP_N, (int)ci, (int)co, (int)k, &one, static_cast<const char*>(ptr(x)) + (b * ci * n + at) * e, type,
            (int)n, (long long)sx, static_cast<const char*>(ptr(gy)) + (b * co * n + at) * e, type, (int)n, (long long)sy, &beta,
            fptr(partial) + b * slices * co * ci, CUDA_R_32F, (int)ci, (long long)(out_step * co * ci), (int)count, compute, CUBLAS_GEMM_DEFAULT);
        TORCH_CHECK(st == CUBLAS_STATUS_SUCCESS, "deconver_b200: projection gradient failed (cuBLAS status ", (int)st, ")");
    };
    if (slices == 1) products(0, 0, n, true, batch, 0.0f);
    else
        for (int64_t b = 0; b < batch; ++b) products(b, 0, length, false, slices, 0.0f);
    if (rest) products(0, slices * length, rest, true, batch, 1.0f);
    if (batch * slices == 1 && !bf16) return partial.view(w.sizes());
    check(ndc_proj_sum((int)(batch * slices), co * ci, dtype_code(gy), fptr(partial), ptr(gw), stream()), ndc_proj_last_error());
    return gw;
}

// ---- the layer -------------------------------------------------------------------------------
struct Config {
    int64_t groups, m, sc;
    double eps;
    int64_t iters, grad_iters, flags;
    bool bf16_params = false;          // filter and bias are bfloat16 values
};

bool bf16_params(const Tensor& h0, const Tensor& bias) {
    return h0.scalar_type() == at::kBFloat16 && (!bias.defined() || bias.scalar_type() == at::kBFloat16);
}

NdcDesc make_desc(const Tensor& x, const Tensor& h0, const Config& c, bool relu) {
    NdcDesc d;
    int64_t sp[3] = {1, 1, 1}, k[3] = {1, 1, 1};
    const int64_t rank = x.dim() - 2;
    for (int64_t i = 0; i < rank; ++i) { sp[3 - rank + i] = x.size(2 + i); k[3 - rank + i] = h0.size(2 + i); }
    d.batch = (int)x.size(0); d.groups = (int)c.groups; d.m = (int)c.m; d.sc = (int)c.sc;
    d.D = (int)sp[0]; d.H = (int)sp[1]; d.W = (int)sp[2];
    d.kD = (int)k[0]; d.kH = (int)k[1]; d.kW = (int)k[2];
    d.eps = (float)c.eps; d.relu_input = relu ? 1 : 0; d.dtype = dtype_code(x); d.flags = (int)c.flags;
    if (c.bf16_params) d.flags |= NDC_FLAG_BF16_PARAMS;
    return d;
}

// relu(h0) and the bias as the kernels take them
void prepare_params(const Tensor& h0, const Tensor& bias, Tensor& h, Tensor& b) {
    const auto f32 = h0.options().dtype(at::kFloat);
    const bool same = !bias.defined() || bias.scalar_type() == h0.scalar_type();
    if (kernel_dtype(h0) && same) {
        h = at::empty(h0.sizes(), f32);
        const bool convert = bias.defined() && bias.scalar_type() != at::kFloat;
        b = convert ? at::empty(bias.sizes(), f32) : bias;
        check(ndc_params_prepare(dtype_code(h0), ptr(h0), h0.numel(), fptr(h), convert ? ptr(bias) : nullptr,
                                 convert ? bias.numel() : 0, convert ? fptr(b) : nullptr, stream()),
              ndc_proj_last_error());
        return;
    }
    h = at::relu(h0).to(at::kFloat);
    b = bias.defined() ? bias.to(at::kFloat) : bias;
}

struct Saved {
    Tensor x;                          // the input, rows padded where that pays
    Tensor h, b;                       // float32 filter and bias
    std::vector<Tensor> z, t1;         // per update that has gradients: its source and K(source)
    int64_t first = 0;                 // index of the first such update
};

Tensor run_forward(const Tensor& x, const Tensor& h0, const Tensor& w, const Tensor& bias, const Config& config,
                   Saved* saved) {
    Saved local;
    Saved& sv = saved ? *saved : local;
    Config c = config;
    c.bf16_params = bf16_params(h0, bias);
    // Without gradients float32 parameters need no pass of their own: the depthwise kernels rectify the
    // filter on load (one launch of three less on a single small image).
    bool raw = !saved && c.m == 1 && c.sc == 4 && h0.scalar_type() == at::kFloat &&
               (!bias.defined() || bias.scalar_type() == at::kFloat) && !(c.flags & NDC_FLAG_FORCE_GENERIC);
    if (raw) { sv.h = h0; sv.b = bias; }
    else prepare_params(h0, bias, sv.h, sv.b);
    auto out_shape = x.sizes().vec();
    out_shape[1] = c.groups * c.sc;
    // Rows that are not whole vectors: the layer owns everything between its input and its output
    // (projection, t1, gradients), so it keeps them with padded rows.  One copy of x (a tenth of
    // the forward's traffic) buys vector loads in every kernel and aligned GEMMs.
    const int W = x.numel() ? (int)x.size(-1) : 0;
    int pitch = W;
    sv.x = x;
    if (x.numel()) {
        const NdcDesc d = make_desc(x, h0, c, true);
        pitch = ndc_row_pitch(&d);
        if (pitch != W) {
            auto xs = x.sizes().vec();
            xs.back() = pitch;
            sv.x = at::empty(xs, x.options());
            check(ndc_pad_rows(x.numel() / W, W, pitch, d.dtype, ptr(x), ptr(sv.x), stream()), ndc_proj_last_error());
        }
    }
    auto shape = out_shape;
    if (W) shape.back() = pitch;
    const int64_t n = sv.x.numel() ? sv.x.numel() / (x.size(0) * x.size(1)) : 0;
    Tensor s = at::empty(shape, x.options());
    channel_gemm(w, false, sv.x, s, x.size(0), n, false);
    sv.first = c.iters > c.grad_iters ? c.iters - c.grad_iters : 0;
    Tensor t1;
    for (int64_t it = 0; it < c.iters; ++it) {
        const bool keep = saved && it >= sv.first;
        const bool last = it + 1 == c.iters;
        Tensor out = at::empty(last ? out_shape : shape, x.options());
        if (keep || !t1.defined()) t1 = at::empty(sv.x.sizes(), x.options());
        if (x.numel()) {
            NdcDesc d = make_desc(x, h0, c, it == 0);
            Span span(0);
            auto update = [&](int flag) {
                d.flags = (int)c.flags | (c.bf16_params ? NDC_FLAG_BF16_PARAMS : 0) | flag;
                return ndc_fwd_rows(&d, pitch, last ? W : pitch, ptr(sv.x), ptr(s), fptr(sv.h), it == 0 ? fptr(sv.b) : nullptr,
                                    ptr(out), ptr(t1), stream());
            };
            int status = update(raw ? NDC_FLAG_RELU_FILTER : 0);
            if (raw && status == NDC_ERR_UNSUPPORTED) {   // not the depthwise kernels
                raw = false;
                prepare_params(h0, bias, sv.h, sv.b);
                status = update(0);
            }
            check(status, ndc_last_error());
        }
        if (keep) { sv.z.push_back(s); sv.t1.push_back(t1); }
        s = out;
    }
    return s;
}

struct LayerNode : public torch::autograd::Function<LayerNode> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& h0, const Tensor& w,
                          const std::optional<Tensor>& bias, int64_t groups, int64_t m, int64_t sc, double eps,
                          int64_t iters, int64_t grad_iters, int64_t flags) {
        const Config c{groups, m, sc, eps, iters, grad_iters, flags};
        Saved sv;
        const Tensor b = bias ? *bias : Tensor();
        Tensor out = run_forward(x, h0, w, b, c, &sv);
        variable_list keep = {sv.x, h0, w, b, sv.h, sv.b};
        keep.insert(keep.end(), sv.z.begin(), sv.z.end());
        keep.insert(keep.end(), sv.t1.begin(), sv.t1.end());
        ctx->save_for_backward(keep);
        auto& d = ctx->saved_data;
        d["cfg"] = std::vector<int64_t>{groups, m, sc, iters, grad_iters, flags, sv.first, x.size(-1)};
        d["eps"] = eps;
        return out;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "double backward through the fused Deconv update is not supported");
        const variable_list kept = ctx->get_saved_variables();
        const auto cfg = ctx->saved_data["cfg"].toIntVector();
        Config c{cfg[0], cfg[1], cfg[2], ctx->saved_data["eps"].toDouble(), cfg[3], cfg[4], cfg[5]};
        const int64_t first = cfg[6], count = c.iters - first, W = cfg[7];
        const Tensor &x = kept[0], &h0 = kept[1], &w = kept[2], &bias = kept[3], &h = kept[4], &b = kept[5];
        c.bf16_params = bf16_params(h0, bias);
        const bool need_x = ctx->needs_input_grad(0), need_h = ctx->needs_input_grad(1);
        const bool whole = first == 0;                   // gradients reach the projection
        const bool need_w = whole && ctx->needs_input_grad(2);
        const bool need_b = whole && bias.defined() && ctx->needs_input_grad(3);
        c10::cuda::CUDAGuard guard(x.device());
        const auto f32 = h.options();

        Tensor g = grads[0].contiguous();
        if (g.scalar_type() != x.scalar_type()) g = g.to(x.scalar_type());
        Tensor gx, gh, gb, ws;
        const int64_t n = x.numel() ? x.numel() / (x.size(0) * x.size(1)) : 0;
        for (int64_t i = count - 1; i >= 0; --i) {
            const Tensor &z = kept[6 + i], &t1 = kept[6 + count + i];
            const bool it0 = first + i == 0;
            const bool need_z = i > 0 || (it0 && (need_x || need_w || need_b));
            Tensor gx_i, gz, gh_i;
            if (need_x) gx_i = at::empty(x.sizes(), x.options());
            if (need_z) gz = at::empty(z.sizes(), z.options());
            if (need_h) gh_i = at::empty(h.sizes(), f32);
            if (need_b && it0) gb = at::empty(bias.sizes(), f32);
            if (x.numel()) {
                NdcDesc d = make_desc(x, h0, c, it0);
                const int pitch = d.W;
                d.W = (int)W;
                const size_t bytes = ndc_bwd_rows_workspace_bytes(&d, pitch);
                if (!ws.defined()) ws = at::empty({(int64_t)bytes}, x.options().dtype(at::kByte));
                Span span(1);
                check(ndc_bwd_rows(&d, pitch, i == count - 1 ? (int)W : pitch, ptr(x), ptr(z), ptr(t1), fptr(h),
                                   it0 ? fptr(b) : nullptr, ptr(g), ptr(gx_i), ptr(gz), fptr(gh_i),
                                   it0 ? fptr(gb) : nullptr, ptr(ws), bytes, stream()), ndc_last_error());
            } else {
                for (Tensor* t : {&gx_i, &gz, &gh_i, &gb}) if (t->defined()) t->zero_();
            }
            if (need_x) { if (gx.defined()) gx.add_(gx_i); else gx = gx_i; }
            if (need_h) { if (gh.defined()) gh.add_(gh_i); else gh = gh_i; }
            g = gz;
        }
        ws.reset();
        Tensor gw, gh0, gbias;
        if (whole) {
            // gz of the first update: W^T gz is added to the update's own input gradient
            if (need_x) channel_gemm(w, true, g, gx, x.size(0), n, true);
            if (need_w) gw = weight_grad(g, x, w, x.size(0), n);
        }
        if (need_x && x.numel() && x.size(-1) != W) {
            auto xs = x.sizes().vec();
            xs.back() = W;
            Tensor plain = at::empty(xs, x.options());
            check(ndc_unpad_rows(plain.numel() / W, (int)W, (int)x.size(-1), dtype_code(x), ptr(gx), ptr(plain), stream()),
                  ndc_proj_last_error());
            gx = plain;
        }
        const bool same = !need_b || !need_h || bias.scalar_type() == h0.scalar_type();
        if ((need_h || need_b) && kernel_dtype(need_h ? h0 : bias) && same) {
            if (need_h) gh0 = at::empty(h0.sizes(), h0.options());
            const bool convert = need_b && bias.scalar_type() != at::kFloat;
            gbias = convert ? at::empty(bias.sizes(), bias.options()) : gb;
            if (need_h || convert)
                check(ndc_params_grad(dtype_code(need_h ? h0 : bias), need_h ? ptr(h0) : nullptr, fptr(gh),
                                      need_h ? h0.numel() : 0, ptr(gh0), convert ? fptr(gb) : nullptr,
                                      convert ? bias.numel() : 0, convert ? ptr(gbias) : nullptr, stream()),
                      ndc_proj_last_error());
        } else {
            if (need_h) gh0 = gh.mul_(h0 > 0).to(h0.scalar_type());
            if (need_b) gbias = gb.to(bias.scalar_type());
        }
        variable_list out(11);
        out[0] = gx; out[1] = gh0; out[2] = gw; out[3] = gbias;
        return out;
    }
};

// s of the layer.  `h0` (C, sc, *k), `w` (groups*sc, C, 1), `bias` (groups*sc) or None.
Tensor layer(const Tensor& x_in, const Tensor& h0_in, const Tensor& w_in, const std::optional<Tensor>& bias_in,
             int64_t groups, int64_t m, int64_t sc, double eps, int64_t iters, int64_t grad_iters, int64_t flags) {
    TORCH_CHECK(w_in.scalar_type() == x_in.scalar_type(), "deconver_b200: the input is ", x_in.scalar_type(),
                " but the projection's weight is ", w_in.scalar_type());
    for (const Tensor* t : {&h0_in, &w_in})
        TORCH_CHECK(t->device() == x_in.device(), "deconver_b200: input on ", x_in.device(), ", parameters on ", t->device());
    TORCH_CHECK(x_in.size(1) == groups * m && w_in.size(0) == groups * sc && w_in.size(1) == x_in.size(1) &&
                h0_in.dim() == x_in.dim() && h0_in.size(0) == groups * m && h0_in.size(1) == sc,
                "deconver_b200: input ", x_in.sizes(), ", filter ", h0_in.sizes(), " and projection ", w_in.sizes(),
                " do not match groups=", groups, ", m=", m, ", sc=", sc);
    TORCH_CHECK(!bias_in || (bias_in->device() == x_in.device() && bias_in->numel() == groups * sc),
                "deconver_b200: the bias does not match the projection");
    c10::cuda::CUDAGuard guard(x_in.device());
    refuse_tangents({&x_in, &h0_in, &w_in});
    if (bias_in) refuse_tangents({&*bias_in});
    const Tensor x = x_in.contiguous(), h0 = h0_in.contiguous(), w = w_in.contiguous();
    const std::optional<Tensor> bias = bias_in ? std::optional<Tensor>(bias_in->contiguous()) : std::nullopt;
    const bool grad = at::GradMode::is_enabled() &&
                      (x.requires_grad() || h0.requires_grad() || w.requires_grad() || (bias && bias->requires_grad()));
    if (grad && grad_iters > 0)
        return LayerNode::apply(x, h0, w, bias, groups, m, sc, eps, iters, grad_iters, flags);
    at::AutoDispatchBelowADInplaceOrView below;
    return run_forward(x, h0, w, bias ? *bias : Tensor(), Config{groups, m, sc, eps, iters, grad_iters, flags}, nullptr);
}

// ---- the layer's neighbours in a block ---------------------------------------------------------
// Small blocks are bound by the host here too: with one Python autograd node each and their parameters
// converted one by one, a training step of a bf16 block of 32 channels x 16^3 took 1.44 - 2.16 ms for
// 0.22 ms of kernels; from here it takes 0.72.  float32 projections lose the convolution route's copies
// to channels-last as well (8 x 32 x 40^3: 11.4 -> 3.4 ms).

// A vector of parameters as float32, and a float32 gradient in the parameters' type: one launch.
Tensor as_f32(const Tensor& t) {
    if (!t.defined() || t.scalar_type() == at::kFloat) return t.defined() ? t.contiguous() : t;
    if (t.scalar_type() != at::kBFloat16 || !t.numel()) return t.to(at::kFloat).contiguous();
    const Tensor in = t.contiguous();
    Tensor out = at::empty(in.sizes(), in.options().dtype(at::kFloat));
    check(ndc_params_prepare(NDC_BF16, nullptr, 0, nullptr, ptr(in), in.numel(), fptr(out), stream()), ndc_proj_last_error());
    return out;
}
Tensor from_f32(const Tensor& g, at::ScalarType type) {
    if (!g.defined() || type == at::kFloat) return g;
    if (type != at::kBFloat16 || !g.numel()) return g.to(type);
    Tensor out = at::empty(g.sizes(), g.options().dtype(type));
    check(ndc_params_grad(NDC_BF16, nullptr, nullptr, 0, nullptr, fptr(g), g.numel(), ptr(out), stream()), ndc_proj_last_error());
    return out;
}

// The gradients of a node whose backward is not itself differentiable: they are computed without a
// graph, and differentiating them raises an error.  What torch.autograd.function.once_differentiable does
// for Python nodes, which these were, message included.
variable_list once(const variable_list& grads, variable_list out) {
    bool any = false;
    for (const Tensor& g : grads) any = any || (g.defined() && g.requires_grad());
    if (!at::GradMode::is_enabled() || !any) return out;
    auto error = std::make_shared<torch::autograd::DelayedError>(
        "trying to differentiate twice a function that was marked with @once_differentiable", (int64_t)out.size());
    for (Tensor& t : out)
        if (t.defined()) t = t.detach().requires_grad_();
    return (*error)(std::move(out));
}

struct Slabs { int batch, channels; int64_t n; };
Slabs slabs(const Tensor& x) {
    const int64_t bc = x.size(0) * x.size(1);
    int64_t n = 1;
    for (int64_t i = 2; i < x.dim(); ++i) n *= x.size(i);
    return {(int)x.size(0), (int)x.size(1), bc ? n : 0};
}
Tensor like(const Tensor& g, const Tensor& x) {
    Tensor c = g.contiguous();
    return c.scalar_type() == x.scalar_type() ? c : c.to(x.scalar_type());
}
Tensor bias_scratch(const Slabs& s, const Tensor& x) {
    return at::empty({(int64_t)ndc_bias_grad_workspace_bytes(s.batch, s.channels)}, x.options().dtype(at::kByte));
}

// y = w x (+ bias) over the channel axis; `w` (Co, Ci, 1)
struct LinearNode : public torch::autograd::Function<LinearNode> {
    static Tensor run(const Tensor& x, const Tensor& w, const Tensor& bias) {
        auto shape = x.sizes().vec();
        shape[1] = w.size(0);
        Tensor y = at::empty(shape, x.options());
        const Slabs s = slabs(y), in = slabs(x);
        if (!y.numel()) return y;
        if (!in.channels) y.zero_();
        else channel_gemm(w, false, x, y, s.batch, s.n, false);
        if (bias.defined()) {
            const Tensor b = as_f32(bias);
            check(ndc_bias_add(s.batch, s.channels, s.n, dtype_code(y), ptr(y), fptr(b), stream()), ndc_bias_last_error());
        }
        return y;
    }

    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const std::optional<Tensor>& bias) {
        const Tensor b = bias ? *bias : Tensor();
        ctx->save_for_backward({x, w});
        ctx->saved_data["bias"] = b.defined();
        ctx->saved_data["type"] = (int64_t)(b.defined() ? b.scalar_type() : at::kFloat);
        return run(x, w, b);
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        variable_list out(3);
        {
            at::AutoGradMode off(false);
            const variable_list kept = ctx->get_saved_variables();
            const Tensor &x = kept[0], &w = kept[1];
            c10::cuda::CUDAGuard guard(x.device());
            const Tensor g = like(grads[0], x);
            const Slabs s = slabs(g);
            if (ctx->needs_input_grad(0)) {
                out[0] = at::empty(x.sizes(), x.options());
                if (s.n) channel_gemm(w, true, g, out[0], s.batch, s.n, false);
                else out[0].zero_();
            }
            if (ctx->needs_input_grad(1)) out[1] = weight_grad(g, x, w, s.batch, s.n);
            if (ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(2)) {
                Tensor gb = at::empty({s.channels}, x.options().dtype(at::kFloat));
                if (s.n) {
                    Tensor ws = bias_scratch(s, x);
                    check(ndc_bias_grad(s.batch, s.channels, s.n, dtype_code(g), ptr(g), fptr(gb), ptr(ws), ws.numel(), stream()),
                          ndc_bias_last_error());
                } else {
                    gb.zero_();
                }
                out[2] = from_f32(gb, (at::ScalarType)ctx->saved_data["type"].toInt());
            }
        }
        return once(grads, out);
    }
};

bool wants_grad(std::initializer_list<const Tensor*> tensors) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : tensors)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}

void check_linear(const Tensor& x_in, const Tensor& w_in, const std::optional<Tensor>& bias_in) {
    TORCH_CHECK(kernel_dtype(x_in) && w_in.scalar_type() == x_in.scalar_type() && w_in.device() == x_in.device() &&
                x_in.dim() >= 3 && w_in.dim() == 3 && w_in.size(2) == 1 && w_in.size(1) == x_in.size(1),
                "deconver_b200: input ", x_in.sizes(), " (", x_in.scalar_type(), ", ", x_in.device(), ") and 1x1 weight ",
                w_in.sizes(), " (", w_in.scalar_type(), ", ", w_in.device(), ") do not match");
    TORCH_CHECK(!bias_in || (bias_in->device() == x_in.device() && bias_in->numel() == w_in.size(0)),
                "deconver_b200: the bias does not match the projection");
}

Tensor linear(const Tensor& x_in, const Tensor& w_in, const std::optional<Tensor>& bias_in) {
    check_linear(x_in, w_in, bias_in);
    c10::cuda::CUDAGuard guard(x_in.device());
    const Tensor x = x_in.contiguous(), w = w_in.contiguous(), b = bias_in ? *bias_in : Tensor();
    refuse_tangents({&x, &w, &b});
    if (wants_grad({&x, &w, &b})) return LinearNode::apply(x, w, bias_in);
    at::AutoDispatchBelowADInplaceOrView below;
    return LinearNode::run(x, w, b);
}

// gelu(h + bias[c]), erf form
struct BiasGeluNode : public torch::autograd::Function<BiasGeluNode> {
    static Tensor run(const Tensor& h, const Tensor& b) {
        Tensor out = at::empty(h.sizes(), h.options());
        const Slabs s = slabs(h);
        if (h.numel())
            check(ndc_bias_gelu_fwd(s.batch, s.channels, s.n, dtype_code(h), ptr(h), fptr(b), ptr(out), stream()), ndc_bias_last_error());
        return out;
    }

    static Tensor forward(AutogradContext* ctx, const Tensor& h, const std::optional<Tensor>& bias) {
        const Tensor b = as_f32(bias ? *bias : Tensor());
        ctx->save_for_backward({h, b});
        ctx->saved_data["bias"] = (int64_t)(bias ? bias->scalar_type() : at::kFloat);
        return run(h, b);
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        variable_list out(2);
        {
            at::AutoGradMode off(false);
            const variable_list kept = ctx->get_saved_variables();
            const Tensor &h = kept[0], &b = kept[1];
            c10::cuda::CUDAGuard guard(h.device());
            const Tensor g = like(grads[0], h);
            const Slabs s = slabs(h);
            const bool want_bias = b.defined() && ctx->needs_input_grad(1);
            out[0] = at::empty(h.sizes(), h.options());
            Tensor gb, ws;
            if (want_bias) {
                gb = at::empty({s.channels}, h.options().dtype(at::kFloat));
                ws = bias_scratch(s, h);
            }
            if (s.n)
                check(ndc_bias_gelu_bwd(s.batch, s.channels, s.n, dtype_code(h), ptr(g), ptr(h), fptr(b), ptr(out[0]), fptr(gb),
                                        ptr(ws), want_bias ? ws.numel() : 0, stream()), ndc_bias_last_error());
            else if (want_bias)
                gb.zero_();
            if (want_bias) out[1] = from_f32(gb, (at::ScalarType)ctx->saved_data["bias"].toInt());
        }
        return once(grads, out);
    }
};

void check_gelu(const Tensor& h_in, const std::optional<Tensor>& bias) {
    TORCH_CHECK(kernel_dtype(h_in) && h_in.is_cuda() && h_in.dim() >= 2 &&
                (!bias || (bias->device() == h_in.device() && bias->numel() == h_in.size(1))),
                "deconver_b200: the bias does not match the tensor");
}

Tensor bias_gelu(const Tensor& h_in, const std::optional<Tensor>& bias) {
    check_gelu(h_in, bias);
    c10::cuda::CUDAGuard guard(h_in.device());
    const Tensor h = h_in.contiguous(), b = bias ? *bias : Tensor();
    refuse_tangents({&h, &b});
    if (wants_grad({&h, &b})) return BiasGeluNode::apply(h, bias);
    at::AutoDispatchBelowADInplaceOrView below;
    return BiasGeluNode::run(h, as_f32(b));
}

// ---- activations and products held in 8 bits ----------------------------------------------------
// Rows of `n` elements as e4m3 values (padded to whole vectors) and the powers of two of their blocks.
struct Held { Tensor values, scales; };

Held empty_held(at::IntArrayRef lead, int64_t n, const Tensor& like) {
    auto v = lead.vec(), s = v;
    v.push_back(ndc_q8_pitch(n));
    s.push_back(ndc_q8_scales(n));
    return {at::empty(v, like.options().dtype(at::kFloat8_e4m3fn)), at::empty(s, like.options().dtype(at::kFloat8_e8m0fnu))};
}
// Blocks along the positions of each (sample, channel), and along the channels of each position (rows then).
Held hold(const Tensor& x) {
    const Slabs s = slabs(x);
    Held h = empty_held({s.batch, s.channels}, s.n, x);
    if (x.numel())
        check(ndc_q8_hold((int64_t)s.batch * s.channels, s.n, dtype_code(x), ptr(x), ptr(h.values), ptr(h.scales), stream()), ndc_q8_last_error());
    return h;
}
// `rows`: where x goes as held along its positions too.
Held hold_channels(const Tensor& x, int64_t batch, int64_t channels, int64_t n, Held* rows = nullptr) {
    Held h = empty_held({batch * n}, channels, x);
    if (rows) *rows = empty_held({batch, channels}, n, x);
    check(ndc_q8_hold_channels((int)batch, (int)channels, n, dtype_code(x), ptr(x), ptr(h.values), ptr(h.scales), rows ? ptr(rows->values) : nullptr,
                               rows ? ptr(rows->scales) : nullptr, stream()), ndc_q8_last_error());
    return h;
}
Tensor read(const Held& h, at::IntArrayRef shape, at::ScalarType type) {
    Tensor x = at::empty(shape, h.values.options().dtype(type));
    const Slabs s = slabs(x);
    if (x.numel())
        check(ndc_q8_read((int64_t)s.batch * s.channels, s.n, dtype_code(x), ptr(h.values), ptr(h.scales), ptr(x), stream()), ndc_q8_last_error());
    return x;
}

std::tuple<Tensor, Tensor> quantize(const Tensor& x_in) {
    TORCH_CHECK(x_in.is_cuda() && kernel_dtype(x_in) && x_in.dim() >= 2, "deconver_b200: quantize takes CUDA float32 / bfloat16 tensors (batch, channels, ...)");
    c10::cuda::CUDAGuard guard(x_in.device());
    refuse_tangents({&x_in});
    at::AutoDispatchBelowADInplaceOrView below;
    const Held h = hold(x_in.contiguous());
    return {h.values, h.scales};
}
Tensor dequantize(const Tensor& values, const Tensor& scales, at::IntArrayRef shape, bool bf16) {
    TORCH_CHECK(shape.size() >= 2, "deconver_b200: dequantize needs a shape (batch, channels, ...)");
    int64_t n = 1;
    for (size_t i = 2; i < shape.size(); ++i) n *= shape[i];
    if (!shape[0] || !shape[1]) n = 0;
    TORCH_CHECK(values.is_cuda() && scales.device() == values.device() && values.scalar_type() == at::kFloat8_e4m3fn &&
                scales.scalar_type() == at::kFloat8_e8m0fnu && values.sizes() == at::IntArrayRef({shape[0], shape[1], ndc_q8_pitch(n)}) &&
                scales.sizes() == at::IntArrayRef({shape[0], shape[1], ndc_q8_scales(n)}),
                "deconver_b200: values ", values.sizes(), " (", values.scalar_type(), ") and scales ", scales.sizes(), " (", scales.scalar_type(),
                ") do not hold a tensor of ", shape);
    c10::cuda::CUDAGuard guard(values.device());
    at::AutoDispatchBelowADInplaceOrView below;
    return read({values.contiguous(), scales.contiguous()}, shape, bf16 ? at::kBFloat16 : at::kFloat);
}

// A bias as the kernels take it: of either type.
Tensor kernel_bias(const Tensor& b) { return !b.defined() || kernel_dtype(b) ? (b.defined() ? b.contiguous() : b) : b.to(at::kFloat).contiguous(); }
int bias_code(const Tensor& b) { return b.defined() ? dtype_code(b) : NDC_F32; }

// out of `rows` neighbours: see ndc_q8_product.  `sum`: over samples, in slices.
void held_product(int64_t samples, int64_t m, int64_t n, int64_t k, const Held& a, const Held& b, const Tensor& bias, int64_t rows, Tensor& out, bool sum) {
    Tensor ws;
    if (sum) ws = at::empty({(int64_t)ndc_q8_product_workspace_bytes((int)samples, m, n, k, dtype_code(out))}, out.options().dtype(at::kByte));
    check(ndc_q8_product((int)samples, m, n, k, dtype_code(out), ptr(a.values), ptr(a.scales), ptr(b.values), ptr(b.scales), ptr(bias), bias_code(bias), rows, ptr(out),
                         ptr(ws), sum ? ws.numel() : 0, stream()), ndc_q8_last_error());
}

// y = w x (+ bias) over the channels of x (batch, ci, n), operands held in 8 bits; `hold_w` gives w as rows of ci.  Up to 512 channels x is
// held on its way to the tensor cores.  `rows`: where x goes as held along its positions, if anywhere.  (x before w: the longer
// launch first, under which the host gets ahead.)
template <class F>
void held_project(const Tensor& x, int64_t batch, int64_t ci, int64_t co, int64_t n, F hold_w, const Tensor& bias, Tensor& y, Held* rows = nullptr) {
    if (ci > 512) {
        const Held h = hold_channels(x, batch, ci, n, rows);
        return held_product(1, batch * n, co, ci, h, hold_w(), bias, n, y, false);
    }
    if (rows) *rows = hold(x);
    const Held w = hold_w();
    check(ndc_q8_project((int)batch, (int)ci, (int)co, n, dtype_code(x), ptr(x), ptr(w.values), ptr(w.scales), ptr(bias), bias_code(bias), ptr(y),
                         stream()), ndc_q8_last_error());
}

// y = w x + bias of bfloat16 tensors, rounded once: the library's product in float32, and a pass that adds the bias, in parts of samples, or of
// a sample's positions.  (Added to a y that is the bias, the library rounds its product first.)  16 x (2048 -> 512) x 4096 142 us, where the
// exact layer, which rounds twice, takes 116; parts of 32 MiB or of all positions take 161 and 142.
Tensor project_once(const Tensor& x, const Tensor& w, const Tensor& bias) {
    constexpr int64_t kMost = 32 << 20;                        // values of a part
    auto shape = x.sizes().vec();
    shape[1] = w.size(0);
    Tensor y = at::empty(shape, x.options());
    const Slabs s = slabs(x);
    const int64_t co = w.size(0), ci = s.channels;
    const auto parts_of = [](int64_t count, int64_t most) { const int64_t parts = (count + most - 1) / most; return (count + parts - 1) / parts; };
    const int64_t samples = parts_of(s.batch, std::max<int64_t>(1, kMost / (co * s.n)));
    const int64_t positions = samples > 1 ? s.n : std::min(s.n, (parts_of(s.n, std::max<int64_t>(128, kMost / co)) + 127) / 128 * 128);
    const Tensor b = as_f32(bias), v = at::empty({samples * co * positions}, x.options().dtype(at::kFloat));
    cublasHandle_t handle = at::cuda::getCurrentCUDABlasHandle();
    const float one = 1.0f, zero = 0.0f;
    for (int64_t i = 0; i < s.batch; i += samples)
        for (int64_t p = 0; p < s.n; p += positions) {
            const int64_t count = std::min(samples, s.batch - i), n = std::min(positions, s.n - p);
            const cublasStatus_t st = cublasGemmStridedBatchedEx(
                handle, CUBLAS_OP_N, CUBLAS_OP_N, (int)n, (int)co, (int)ci, &one, static_cast<const at::BFloat16*>(ptr(x)) + i * ci * s.n + p, CUDA_R_16BF,
                (int)s.n, (long long)(ci * s.n), ptr(w), CUDA_R_16BF, (int)ci, 0LL, &zero, ptr(v), CUDA_R_32F, (int)n, (long long)(co * n), (int)count,
                CUBLAS_COMPUTE_32F, CUBLAS_GEMM_DEFAULT);
            TORCH_CHECK(st == CUBLAS_STATUS_SUCCESS, "deconver_b200: projection GEMM failed (cuBLAS status ", (int)st, ")");
            check(ndc_bias_round((int)count, (int)co, n, fptr(v), fptr(b), static_cast<at::BFloat16*>(ptr(y)) + i * co * s.n + p, s.n, stream()), ndc_bias_last_error());
        }
    return y;
}

// Where the weight gradient of a checkpoint is the library's product after all, of what is read back: large bfloat16 products, whose
// held operand ndc_q8_wgrad decodes once for each 128 outputs.  Microseconds, ndc_q8_wgrad and the other way, at batch x (inputs ->
// outputs) x positions: 16 x (512 -> 2048) x 4096 298 and 224, 16 x (256 -> 1024) x 16384 283 and 256, 4 x (2048 -> 2048) x 8192
// 575 and 264; but 16 x (256 -> 1024) x 4096 89 and 110, 8 x (1024 -> 1024) x 1000 60 and 79, 2 x (64 -> 256) x 262144 66 and 150.
// (All of what is read back is in memory meanwhile, a bfloat16 copy of the input.)  Rows of whole vectors only: for others the library has its
// convolution, whose sums need not come in the same order every time, and which is the slower one: 1 x (512 -> 512) x 200003 641 us for 1006,
// 4 x (512 -> 512) x 100003 1266 for 4483, 16 x (512 -> 2048) x 4095 707 for 1098 (with the bias gradient).
bool library_wgrad(const Tensor& g, int64_t co, int64_t ci, int64_t batch, int64_t n) {
    return g.scalar_type() == at::kBFloat16 && n % 8 == 0 && co * ci >= 1 << 18 && 2.0 * (double)batch * (double)n * (double)(co * ci) >= 1e11;
}

// y = w x (+ bias); what the backward knows of x is held in 8 bits.  `products`: those of operands held in 8 bits, each in
// blocks along what it is summed over.
struct HeldLinearNode : public torch::autograd::Function<HeldLinearNode> {
    // `held`: x in 8 bits for the backward, or nothing
    static Tensor run(const Tensor& x, const Tensor& w, const Tensor& bias, bool products, Held* held) {
        auto shape = x.sizes().vec();
        shape[1] = w.size(0);
        const Slabs in = slabs(x);
        const int64_t co = w.size(0);
        // bfloat16 rows and weights of whole vectors: one pass that holds x.  Where w does not fit it whole, in parts if there is a bias, else the
        // library's product, which is rounded once without one: with the pass that holds x 14, 32 and 136 us for 14, 41 and 236 at 2 x and 16 x
        // (512 -> 2048) x 512 and 16 x (512 -> 2048) x 4096.  (With a bias 14, 41 and 236 for 26, 74 and 228 of the exact layer's launches.)
        const bool whole = !products && in.n && co && x.scalar_type() == at::kBFloat16 && in.n % 8 == 0 && in.channels % 8 == 0;
        if (whole && ((uintptr_t)ptr(x) | (uintptr_t)ptr(w)) % 16 == 0) {
            const bool one = ndc_q8_linear_fwd_applies(in.batch, in.channels, (int)co, in.n);
            if (one || (bias.defined() && ndc_q8_linear_fwd_parts_applies(in.batch, in.channels, (int)co, in.n))) {
                Tensor y = at::empty(shape, x.options());
                if (held) *held = empty_held({in.batch, in.channels}, in.n, x);
                const Tensor b = kernel_bias(bias);
                check((one ? ndc_q8_linear_fwd : ndc_q8_linear_fwd_parts)(in.batch, in.channels, (int)co, in.n, ptr(x), ptr(w), ptr(b), bias_code(b), ptr(y),
                                                                           held ? ptr(held->values) : nullptr, held ? ptr(held->scales) : nullptr, stream()),
                      ndc_q8_last_error());
                return y;
            }
        }
        if (!products || !in.n || !co) {
            if (held) *held = hold(x);
            // (ragged positions or channels: the exact layer's result, to the bit)
            return whole && bias.defined() ? project_once(x, w, bias) : LinearNode::run(x, w, bias);
        }
        Tensor y = at::empty(shape, x.options());
        held_project(x, in.batch, in.channels, co, in.n, [&] { return hold(w.view({1, co, w.size(1)})); }, kernel_bias(bias), y, held);
        return y;
    }

    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const std::optional<Tensor>& bias, bool products) {
        const Tensor b = bias ? *bias : Tensor();
        Held h;
        Tensor y = run(x, w, b, products, w.requires_grad() ? &h : nullptr);       // no other gradient asks for it
        ctx->save_for_backward({h.values, h.scales, w});
        auto& d = ctx->saved_data;
        d["shape"] = x.sizes().vec();
        d["products"] = products;
        d["bias"] = b.defined();
        d["type"] = (int64_t)(b.defined() ? b.scalar_type() : at::kFloat);
        return y;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        variable_list out(4);
        {
            at::AutoGradMode off(false);
            const variable_list kept = ctx->get_saved_variables();
            const Held held{kept[0], kept[1]};
            const Tensor& w = kept[2];
            auto& d = ctx->saved_data;
            const std::vector<int64_t> shape = d["shape"].toIntVector();
            const bool products = d["products"].toBool();
            c10::cuda::CUDAGuard guard(w.device());
            const Tensor g = like(grads[0], w);
            const Slabs s = slabs(g);
            const int64_t ci = shape[1], co = w.size(0);
            if (ctx->needs_input_grad(0)) {
                out[0] = at::empty(shape, g.options());
                if (!s.n || !ci) out[0].zero_();
                else if (!products) channel_gemm(w, true, g, out[0], s.batch, s.n, false);
                else held_project(g, s.batch, co, ci, s.n, [&] { return hold_channels(w, 1, co, ci); }, Tensor(), out[0]);
            }
            if (ctx->needs_input_grad(1)) {
                if (!s.n || !ci || !co) out[1] = at::zeros(w.sizes(), w.options());
                else {
                    // the bias gradient from the same pass over g
                    const auto type = (at::ScalarType)d["type"].toInt();
                    const bool library = !products && library_wgrad(g, co, ci, s.batch, s.n);
                    out[1] = library ? weight_grad(g, read(held, shape, g.scalar_type()), w, s.batch, s.n) : at::empty(w.sizes(), w.options());
                    const bool bias = !library && d["bias"].toBool() && ctx->needs_input_grad(2) && (type == at::kFloat || type == at::kBFloat16);
                    const int code = type == at::kBFloat16 ? NDC_BF16 : NDC_F32;
                    if (bias) out[2] = at::empty({co}, g.options().dtype(type));
                    if (products) {
                        Held h;
                        if (bias) {
                            h = empty_held({s.batch, s.channels}, s.n, g);
                            Tensor ws = bias_scratch(s, g);
                            check(ndc_q8_hold_sum(s.batch, s.channels, s.n, dtype_code(g), ptr(g), ptr(h.values), ptr(h.scales), ptr(out[2]), code, ptr(ws),
                                                  ws.numel(), stream()), ndc_q8_last_error());
                        } else {
                            h = hold(g);
                        }
                        held_product(s.batch, ci, co, s.n, held, h, Tensor(), ci, out[1], true);
                    } else if (!library) {
                        const size_t bytes = ndc_q8_wgrad_workspace_bytes(s.batch, (int)co, (int)ci, s.n, dtype_code(g));
                        Tensor ws = at::empty({(int64_t)bytes}, g.options().dtype(at::kByte));
                        check(ndc_q8_wgrad(s.batch, (int)co, (int)ci, s.n, dtype_code(g), ptr(g), ptr(held.values), ptr(held.scales), ptr(out[1]), ptr(out[2]),
                                           code, ptr(ws), bytes, stream()), ndc_q8_last_error());
                    }
                }
            }
            if (d["bias"].toBool() && ctx->needs_input_grad(2) && !out[2].defined()) {
                Tensor gb = at::empty({s.channels}, g.options().dtype(at::kFloat));
                if (s.n) {
                    Tensor ws = bias_scratch(s, g);
                    check(ndc_bias_grad(s.batch, s.channels, s.n, dtype_code(g), ptr(g), fptr(gb), ptr(ws), ws.numel(), stream()),
                          ndc_bias_last_error());
                } else {
                    gb.zero_();
                }
                out[2] = from_f32(gb, (at::ScalarType)d["type"].toInt());
            }
        }
        return once(grads, out);
    }
};

Tensor linear_q8(const Tensor& x_in, const Tensor& w_in, const std::optional<Tensor>& bias_in, bool products) {
    check_linear(x_in, w_in, bias_in);
    TORCH_CHECK(!products || slabs(x_in).n <= 1 << 24, "deconver_b200: products in 8 bits take inputs of up to 2^24 positions per sample, not ", x_in.sizes());
    c10::cuda::CUDAGuard guard(x_in.device());
    const Tensor x = x_in.contiguous(), w = w_in.contiguous(), b = bias_in ? *bias_in : Tensor();
    refuse_tangents({&x, &w, &b});
    if (wants_grad({&x, &w, &b})) return HeldLinearNode::apply(x, w, bias_in, products);
    at::AutoDispatchBelowADInplaceOrView below;
    return HeldLinearNode::run(x, w, b, products, nullptr);
}

// gelu(h + bias[c]); the backward knows h as it is held in 8 bits
struct HeldGeluNode : public torch::autograd::Function<HeldGeluNode> {
    static Tensor run(const Tensor& h, const Tensor& b, const Held& held) {
        Tensor out = at::empty(h.sizes(), h.options());
        const Slabs s = slabs(h);
        if (h.numel())
            check(ndc_q8_bias_gelu_fwd(s.batch, s.channels, s.n, dtype_code(h), ptr(h), fptr(b), ptr(out), ptr(held.values), ptr(held.scales), stream()),
                  ndc_q8_last_error());
        return out;
    }

    static Tensor forward(AutogradContext* ctx, const Tensor& h, const std::optional<Tensor>& bias) {
        const Tensor b = as_f32(bias ? *bias : Tensor());
        const Slabs s = slabs(h);
        const Held held = empty_held({s.batch, s.channels}, s.n, h);
        Tensor out = run(h, b, held);
        ctx->save_for_backward({held.values, held.scales, b});
        ctx->saved_data["bias"] = (int64_t)(bias ? bias->scalar_type() : at::kFloat);
        ctx->saved_data["type"] = (int64_t)h.scalar_type();
        return out;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        variable_list out(2);
        {
            at::AutoGradMode off(false);
            const variable_list kept = ctx->get_saved_variables();
            const Tensor &values = kept[0], &b = kept[2];
            c10::cuda::CUDAGuard guard(values.device());
            Tensor g = grads[0].contiguous();
            const auto type = (at::ScalarType)ctx->saved_data["type"].toInt();
            if (g.scalar_type() != type) g = g.to(type);
            const Slabs s = slabs(g);
            const bool want_bias = b.defined() && ctx->needs_input_grad(1);
            out[0] = at::empty(g.sizes(), g.options());
            Tensor gb, ws;
            if (want_bias) {
                gb = at::empty({s.channels}, g.options().dtype(at::kFloat));
                ws = bias_scratch(s, g);
            }
            if (s.n)
                check(ndc_q8_bias_gelu_bwd(s.batch, s.channels, s.n, dtype_code(g), ptr(g), ptr(values), ptr(kept[1]), fptr(b), ptr(out[0]), fptr(gb),
                                           ptr(ws), want_bias ? ws.numel() : 0, stream()), ndc_q8_last_error());
            else if (want_bias)
                gb.zero_();
            if (want_bias) out[1] = from_f32(gb, (at::ScalarType)ctx->saved_data["bias"].toInt());
        }
        return once(grads, out);
    }
};

Tensor bias_gelu_q8(const Tensor& h_in, const std::optional<Tensor>& bias) {
    check_gelu(h_in, bias);
    c10::cuda::CUDAGuard guard(h_in.device());
    const Tensor h = h_in.contiguous(), b = bias ? *bias : Tensor();
    refuse_tangents({&h, &b});
    if (wants_grad({&h, &b})) return HeldGeluNode::apply(h, bias);
    at::AutoDispatchBelowADInplaceOrView below;
    return HeldGeluNode::run(h, as_f32(b), Held());
}

// (x - mean) / sqrt(var + eps) [* weight + bias] per (sample, channel)
struct NormNode : public torch::autograd::Function<NormNode> {
    static Tensor run(const Tensor& x, const Tensor& w, const Tensor& b, double eps, Tensor& stats) {
        Tensor y = at::empty(x.sizes(), x.options());
        const Slabs s = slabs(x);
        stats = at::empty({(int64_t)s.batch * s.channels * 2}, x.options().dtype(at::kFloat));
        if (x.numel()) {
            const size_t bytes = ndc_inorm_workspace_bytes(s.batch, s.channels);
            Tensor ws = at::empty({(int64_t)bytes}, x.options().dtype(at::kByte));
            check(ndc_inorm_fwd(s.batch, s.channels, s.n, dtype_code(x), ptr(x), fptr(w), fptr(b), (float)eps, ptr(y), fptr(stats),
                                ptr(ws), bytes, stream()), ndc_inorm_last_error());
        }
        return y;
    }

    static Tensor forward(AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& weight,
                          const std::optional<Tensor>& bias, double eps) {
        const Tensor w = weight ? *weight : Tensor();
        Tensor stats;
        Tensor y = run(x, as_f32(w), as_f32(bias ? *bias : Tensor()), eps, stats);
        ctx->save_for_backward({x, w, stats});
        // a bias without a weight keeps its gradient in float32
        ctx->saved_data["type"] = (int64_t)(w.defined() ? w.scalar_type() : at::kFloat);
        ctx->saved_data["bias"] = bias.has_value();
        return y;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        variable_list out(4);
        {
            at::AutoGradMode off(false);
            const variable_list kept = ctx->get_saved_variables();
            const Tensor &x = kept[0], &w = kept[1], &stats = kept[2];
            c10::cuda::CUDAGuard guard(x.device());
            const Tensor g = like(grads[0], x);
            const Slabs s = slabs(x);
            const auto f32 = x.options().dtype(at::kFloat);
            Tensor gx = at::empty(x.sizes(), x.options()), gw, gb;
            if (w.defined() && ctx->needs_input_grad(1)) gw = at::empty({s.channels}, f32);
            // (gradients are counted over the tensors that are there)
            if (ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(w.defined() ? 2 : 1)) gb = at::empty({s.channels}, f32);
            if (x.numel()) {
                const Tensor wf = as_f32(w);
                const size_t bytes = ndc_inorm_workspace_bytes(s.batch, s.channels);
                Tensor ws = at::empty({(int64_t)bytes}, x.options().dtype(at::kByte));
                check(ndc_inorm_bwd(s.batch, s.channels, s.n, dtype_code(x), ptr(x), ptr(g), fptr(wf), fptr(stats), ptr(gx), fptr(gw),
                                    fptr(gb), ptr(ws), bytes, stream()), ndc_inorm_last_error());
            } else {
                for (Tensor* t : {&gw, &gb}) if (t->defined()) t->zero_();
            }
            const auto type = (at::ScalarType)ctx->saved_data["type"].toInt();
            if (ctx->needs_input_grad(0)) out[0] = gx;
            out[1] = from_f32(gw, type);
            out[2] = from_f32(gb, type);
        }
        return once(grads, out);
    }
};

Tensor instance_norm(const Tensor& x_in, const std::optional<Tensor>& weight, const std::optional<Tensor>& bias, double eps) {
    for (const auto* t : {&weight, &bias})
        TORCH_CHECK(!*t || ((*t)->device() == x_in.device() && (*t)->numel() == x_in.size(1)),
                    "deconver_b200: instance norm parameters do not match the input ", x_in.sizes());
    c10::cuda::CUDAGuard guard(x_in.device());
    const Tensor x = x_in.contiguous(), w = weight ? *weight : Tensor(), b = bias ? *bias : Tensor();
    refuse_tangents({&x, &w, &b});
    if (wants_grad({&x, &w, &b})) return NormNode::apply(x, weight, bias, eps);
    at::AutoDispatchBelowADInplaceOrView below;
    Tensor stats;
    return NormNode::run(x, as_f32(w), as_f32(b), eps, stats);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, mod) {
    mod.def("layer", &layer, py::call_guard<py::gil_scoped_release>());
    mod.def("linear", &linear, py::call_guard<py::gil_scoped_release>());
    mod.def("bias_gelu", &bias_gelu, py::call_guard<py::gil_scoped_release>());
    mod.def("linear_q8", &linear_q8, py::call_guard<py::gil_scoped_release>());
    mod.def("bias_gelu_q8", &bias_gelu_q8, py::call_guard<py::gil_scoped_release>());
    mod.def("quantize", &quantize, py::call_guard<py::gil_scoped_release>());
    mod.def("dequantize", [](const Tensor& values, const Tensor& scales, const std::vector<int64_t>& shape, bool bf16) {
        return dequantize(values, scales, shape, bf16);
    }, py::call_guard<py::gil_scoped_release>());
    mod.def("instance_norm", &instance_norm, py::call_guard<py::gil_scoped_release>());
    mod.def("weight_grad_route", [](int64_t batch, int64_t co, int64_t ci, int64_t n, bool bf16, bool exact, int sms) {
        return (int)plan_weight_grad(batch, co, ci, n, bf16, exact, sms).route;
    });
    mod.def("timing_enable", &timing_enable);
    mod.def("timing_collect", &timing_collect);
}
