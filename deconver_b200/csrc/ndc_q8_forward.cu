// A 1x1 projection of bfloat16 tensors and its input's checkpoint in one pass over the input:
//
//     y[b, o, p] = sum over c of w[o, c] x[b, c, p] (+ bias[o]),   and x held in blocks of 128 positions (ndc_q8.cuh)
//
// The product is that of the bfloat16 operands, summed in float32 and rounded once, the bias in it; the
// library's product, a pass for the bias and one that holds x read y twice more and x once more.
//
// A persistent CTA takes 128 positions of a sample after another.  w stays in shared memory (K-major); blocks of 64 channels
// x 128 positions come by TMA as they lie, positions along the rows of 128 bytes: the MN-major operand of the MMA, and the
// rows that eight warps hold in 8 bits.  The rows of the product are y's channels: a thread that reads one from TMEM has
// neighbouring positions, and writes 16 bytes of them at a time into shared memory, from where they go out by TMA (with
// positions as rows it stored 2 bytes for every four instructions: 78 us at 2 x (64 -> 256) x 64^3).  Two groups of
// four warps do that, of one accumulator while the next is being computed (up to 256 channels: two of them fit).  What bounds it:
// the bytes of x, y and what is held, 370 MB in 66 us there (5.6 TB/s).
//
// A w that does not fit goes in parts of 128 to 512 outputs, CTAs each; those of a tile run at the same time, have x from the L2
// cache, and hold a part of its blocks each.  2 x (64 -> 1024) x 64^3 252 us; 16 x (512 -> 2048) x 4096 236, bound by x's 1.1 GB out of the
// L2 cache and 16 parts of nine CTAs.
#include <algorithm>

#include "ndc_b200.h"
#include "ndc_common.cuh"
#include "ndc_q8_host.h"
#include "ndc_q8_mma.cuh"
#include "ndc_slab.cuh"
#include "ndc_tc_host.h"

namespace ndc {
namespace q8 {
namespace {

typedef __nv_bfloat16 bf16;

constexpr int kStoreWarps = 8, kHoldWarps = 8;
constexpr int kThreads = 32 * (kStoreWarps + kHoldWarps + 2);
constexpr int KC = 64;                       // channels of a block
constexpr int kHalf = KC * 128;              // bytes of 64 positions of a block
constexpr int kBlockBytes = 2 * kHalf;
constexpr int kStaged = MT * 128;            // bytes of 128 channels x 64 positions of y
constexpr int kGaveUp = 480, kBias = 512, kHeader = 4096, kMostSlots = 12;         // barriers, the bias as float32, operands
constexpr int kMostWeights = 128 * 1024;     // bytes of w in shared memory
constexpr int kRoom = 227 * 1024 - 1024 - kHeader;

struct ForwardArgs {
    const void* bias;                        // float32, or bfloat16, or NULL
    int bias_bf16;
    unsigned char *values, *scales;          // or NULL
    long long n, pitch;
    int scale_pitch;
    int ci, co, blocks, columns;             // blocks of input channels; outputs of a part as the MMA takes them, a multiple of 128
    int tiles_n, tiles;                      // of a sample, of all
    int slots, buffers, staged;              // blocks of x in shared memory, accumulators, and places for results of a group
    unsigned* expired;
};

__device__ __forceinline__ void tma_load3(unsigned dst, const CUtensorMap* map, int x, int y, int z, unsigned bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}
__device__ __forceinline__ void group_sync(int group) { asm volatile("bar.sync %0, 128;" ::"r"(1 + group) : "memory"); }
// MN-major rows of 64 positions (128 bytes, swizzled): kHalf to the next 64 positions, 1024 bytes to the next eight channels.
__device__ __forceinline__ unsigned long long positions_desc(unsigned addr) {
    return (unsigned long long)((addr >> 4) & 0x3fff) | (unsigned long long)(kHalf >> 4) << 16 | (unsigned long long)(1024 >> 4) << 32 | 1ull << 46 |
           2ull << 61;
}

// PARTS: of the outputs, in the grid's y.  (One part by the same code took 2 - 4 % more: 167 us for 161 at 2 x (256 -> 64) x 64^3.)
template <bool PARTS>
__global__ void __launch_bounds__(kThreads, 1) forward_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                                                              const __grid_constant__ CUtensorMap map_y, const __grid_constant__ ForwardArgs P) {
    extern __shared__ unsigned char raw_smem[];
    unsigned char* smem = raw_smem + ((1024u - (smem_u32(raw_smem) & 1023u)) & 1023u);
    const unsigned base = smem_u32(smem);
    const unsigned full = base, empty = full + 8 * kMostSlots, dfull = empty + 8 * kMostSlots, dempty = dfull + 16, wfull = dempty + 16, slot_at = wfull + 8;
    const int weights = P.blocks * P.columns * 128;                       // bytes
    const unsigned w_at = base + kHeader, y_at = w_at + weights, x_at = y_at + 2 * P.staged * kStaged;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int o0 = PARTS ? blockIdx.y * P.columns : 0;                    // the part's first output
    if (threadIdx.x == 0) {
        for (int i = 0; i < P.slots; ++i) { mbar_init(full + 8 * i, 1); mbar_init(empty + 8 * i, 1 + (P.values ? kHoldWarps : 0)); }
        for (int i = 0; i < 2; ++i) { mbar_init(dfull + 8 * i, 1); mbar_init(dempty + 8 * i, kStoreWarps); }
        mbar_init(wfull, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (threadIdx.x < 2) reinterpret_cast<volatile unsigned*>(smem + kGaveUp)[threadIdx.x] = 0u;
    if (warp == 0) tmem_alloc(slot_at, 512);
    for (int j = threadIdx.x; j < (kHeader - kBias) / 4; j += kThreads) reinterpret_cast<float*>(smem + kBias)[j] = P.bias && (!PARTS || j < P.columns) && o0 + j < P.co ? load_bias(P.bias, P.bias_bf16, o0 + j) : 0.0f;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const unsigned tmem = *reinterpret_cast<volatile unsigned*>(smem + (slot_at - base));
    bool ok = true;

    if (warp < kStoreWarps) {
        // units of 128 channels x 64 positions, every second one a group's; a thread has a channel
        const int quarter = warp & 3, group = warp >> 2, row = 32 * quarter + lane, units = P.columns / MT * 2;
        const float* bias = reinterpret_cast<const float*>(smem + kBias);
        const bool copies = quarter == 0 && lane == 0;
        // a group whose wait ran out, as seen by all of it after its next barrier: it leaves together
        volatile unsigned* const gave_up = reinterpret_cast<volatile unsigned*>(smem + kGaveUp) + group;
        int count = 0, place = 0;
        for (int t = blockIdx.x; t < P.tiles && ok; t += gridDim.x, ++count) {
            const int sample = t / P.tiles_n, d = count % P.buffers, p = (t - sample * P.tiles_n) * MT;
            if (!mbar_wait(dfull + 8 * d, (count / P.buffers) & 1)) { ok = false; *gave_up = 1u; }
            tc_fence_after();
            for (int u = group; u < units; u += 2) {
                const unsigned acc = tmem + ((unsigned)(32 * quarter) << 16) + d * 256 + u * 64;
                unsigned char* to = smem + (y_at - base) + (group * P.staged + place) * kStaged + row * 128;
                const float b = bias[u / 2 * MT + row];
                // the place is free where its last copy has read it
                if (copies) { if (P.staged == 2) copies_read<1>(); else copies_read<0>(); }
                group_sync(group);
                if (*gave_up) { ok = false; break; }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float v[32];
                    tmem_load32(acc + 32 * h, v);
#pragma unroll
                    for (int m = 0; m < 4; ++m) {
                        unsigned w[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const __nv_bfloat162 q = __floats2bfloat162_rn(v[8 * m + 2 * i] + b, v[8 * m + 2 * i + 1] + b);
                            w[i] = *reinterpret_cast<const unsigned*>(&q);
                        }
                        *reinterpret_cast<uint4*>(to + (((4 * h + m) ^ (row & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
                if (u + 2 >= units) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(dempty + 8 * d);
                }
                fence_async_proxy();
                group_sync(group);
                const int o = o0 + u / 2 * MT;
                if (copies) tma_store3(&map_y, p + (u & 1) * 64, o, sample, y_at + (group * P.staged + place) * kStaged, p + (u & 1) * 64 < P.n && (!PARTS || o < P.co));
                if (++place == P.staged) place = 0;
            }
        }
        if (copies) copies_done();
    } else if (warp < kStoreWarps + kHoldWarps) {
        // sixteen lanes have a channel's 128 positions; the parts take the blocks in turn
        const int w = warp - kStoreWarps, l = lane & 15, piece = l & 7;
        int slot = 0, phase = 0;
        for (int t = blockIdx.x; P.values && t < P.tiles && ok; t += gridDim.x) {
            const int sample = t / P.tiles_n, k = t - sample * P.tiles_n;
            const long long p = (long long)k * kBlock + 8 * l;
            [[maybe_unused]] unsigned turn = PARTS ? (unsigned)t % gridDim.y * P.blocks % gridDim.y : 0;      // the part that has the tile's first block
            for (int block = 0; block < P.blocks; ++block) {
                ok = mbar_wait(full + 8 * slot, phase);
                if (!ok) break;
                if constexpr (PARTS) {
                    const bool mine = turn == blockIdx.y;
                    if (++turn == gridDim.y) turn = 0;
                    if (!mine) {
                        if (lane == 0) mbar_arrive(empty + 8 * slot);
                        if (++slot == P.slots) { slot = 0; phase ^= 1; }
                        continue;
                    }
                }
                const unsigned char* from = smem + (x_at - base) + slot * kBlockBytes + (l >> 3) * kHalf;
                uint4 q[KC / (2 * kHoldWarps)];
#pragma unroll
                for (int i = 0; i < KC / (2 * kHoldWarps); ++i) {
                    const int c = 2 * (w + kHoldWarps * i) + (lane >> 4);
                    q[i] = *reinterpret_cast<const uint4*>(from + c * 128 + ((piece ^ (c & 7)) << 4));
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(empty + 8 * slot);
#pragma unroll
                for (int i = 0; i < KC / (2 * kHoldWarps); ++i) {
                    const int c = block * KC + 2 * (w + kHoldWarps * i) + (lane >> 4);
                    float v[8];
                    slab::Vec16<bf16>::unpack(q[i], v);
                    unsigned top = larger_magnitudes(larger_magnitudes(q[i].x, q[i].y), larger_magnitudes(q[i].z, q[i].w));
                    top = max(top << 16 & 0x7fffffffu, top & 0x7fff0000u);
#pragma unroll
                    for (int off = 8; off > 0; off >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, off));
                    if (__any_sync(0xffffffffu, top >= kInfinite)) {       // the largest of the finite ones; the others become NaN
                        top = 0u;
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const unsigned m = magnitude(v[j]);
                            if (m < kInfinite) top = max(top, m);
                            else v[j] = __uint_as_float(0x7fffffffu);
                        }
#pragma unroll
                        for (int off = 8; off > 0; off >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, off));
                    }
                    if (c >= P.ci) continue;
                    const unsigned byte = scale_byte(top);
                    const unsigned long long inv = both(scale_inverse(byte));
                    const long long row = (long long)sample * P.ci + c;
                    if (p < P.pitch)
                        *reinterpret_cast<uint2*>(P.values + row * P.pitch + p) =
                            make_uint2(encode4(v[0], v[1], v[2], v[3], inv), encode4(v[4], v[5], v[6], v[7], inv));
                    unsigned char* scales = P.scales + row * P.scale_pitch + k;
                    if (l == 0) *scales = (unsigned char)byte;
                    else if (k == P.tiles_n - 1 && l < P.scale_pitch - k) scales[l] = 1;         // what is never looked at
                }
                if (++slot == P.slots) { slot = 0; phase ^= 1; }
            }
        }
    } else if (warp == kStoreWarps + kHoldWarps) {
        if (lane == 0) {
            expect_bytes(wfull, weights);
            for (int block = 0; block < P.blocks; ++block)
                for (int o = 0; o < P.columns; o += 16) tma_load(w_at + (block * P.columns + o) * 128, &map_w, block * KC, o0 + o, wfull);
            int issued = 0;
            for (int t = blockIdx.x; t < P.tiles && ok; t += gridDim.x) {
                const int sample = t / P.tiles_n, p = (t - sample * P.tiles_n) * MT;
                for (int block = 0; block < P.blocks; ++block, ++issued) {
                    const int s = issued % P.slots;
                    if (issued >= P.slots) ok = mbar_wait_thread(empty + 8 * s, (issued / P.slots - 1) & 1, kWaitLimit);
                    if (!ok) break;
                    expect_bytes(full + 8 * s, kBlockBytes);
                    for (int h = 0; h < 2; ++h) tma_load3(x_at + s * kBlockBytes + h * kHalf, &map_x, p + 64 * h, block * KC, sample, full + 8 * s);
                }
            }
            // copies that nobody may have waited for
            ok = mbar_wait_thread(wfull, 0, kWaitLimit) && ok;
            if (!ok)
                for (int i = max(0, issued - P.slots); i < issued; ++i) mbar_wait_thread(full + 8 * (i % P.slots), (i / P.slots) & 1, kWaitLimit);
        }
    } else {
        if (elect()) {
            int slot = 0, phase = 0, count = 0;
            ok = mbar_wait_thread(wfull, 0, kWaitLimit);
            for (int t = blockIdx.x; t < P.tiles && ok; t += gridDim.x, ++count) {
                const int d = count % P.buffers;
                if (count >= P.buffers) ok = mbar_wait_thread(dempty + 8 * d, (count / P.buffers - 1) & 1, kWaitLimit);
                if (!ok) break;
                for (int block = 0; block < P.blocks; ++block) {
                    ok = mbar_wait_thread(full + 8 * slot, phase, kWaitLimit);
                    if (!ok) break;
                    tc_fence_after();
                    const unsigned long long x = positions_desc(x_at + slot * kBlockBytes);
                    const int steps = (P.ci - block * KC + 15) / 16;
                    {
#pragma unroll
                        for (int m0 = 0; m0 < 512; m0 += MT) {
                            if (m0 >= P.columns) break;
                            const unsigned long long w = swizzled_desc(w_at + (block * P.columns + m0) * 128);
#pragma unroll
                            for (int i = 0; i < KC / 16; ++i)
                                if (i < steps) mma(tmem + d * 256 + m0, w + 2 * i, x + 128 * i, instr_desc(MT) | 1u << 16, block > 0 || i > 0);
                        }
                        mma_commit(empty + 8 * slot);
                        if (block == P.blocks - 1) mma_commit(dfull + 8 * d);
                    }
                    if (++slot == P.slots) { slot = 0; phase ^= 1; }
                }
            }
        }
    }
    if (!ok) report_expired(P.expired);
    __syncwarp();
    __syncthreads();
    if (warp == 0) {
        tc_fence_after();
        tmem_free(tmem, 512);
    }
}

// (co, ci), boxes of 16 rows of 64 channels.
bool make_weight_map(CUtensorMap& map, const void* w, int co, int ci) {
    const EncodeTiled fn = encode_tiled();
    const cuuint64_t dims[2] = {(cuuint64_t)ci, (cuuint64_t)co}, strides[1] = {(cuuint64_t)(2 * ci)};
    const cuuint32_t boxes[2] = {KC, 16}, ones[2] = {1, 1};
    return fn && fn(&map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(w), dims, strides, boxes, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int weight_bytes(int ci, int co) { return (ci + KC - 1) / KC * ((co + MT - 1) / MT * MT) * 128; }

bool fits_positions(int batch, long long n) { return batch > 0 && n > 0 && n % 8 == 0 && n <= (1LL << 25) && (n + MT - 1) / MT <= (0x7fffffffLL - 1024) / batch; }

// Parts of the outputs whose w fits shared memory, as wide as each other.
struct Parts { int columns, parts; };
Parts plan_parts(int ci, int co) {
    const int most = std::min(512, kMostWeights / (128 * ((ci + KC - 1) / KC)) / MT * MT);
    const int parts = (co + most - 1) / most;
    return {((co + parts - 1) / parts + MT - 1) / MT * MT, parts};
}

// CTAs of a part: those of the least rounds of CTAs times tiles.
int ctas_of(int tiles, int parts) {
    const long long sms = ndc::num_sms();
    long long best = 1, best_time = 1LL << 62;
    for (long long ctas : {sms / parts, (sms + parts - 1) / parts}) {
        ctas = std::max(1LL, std::min(ctas, (long long)tiles));
        const long long time = (ctas * parts + sms - 1) / sms * ((tiles + ctas - 1) / ctas);
        if (time < best_time) { best_time = time; best = ctas; }
    }
    return (int)best;
}

int check_forward(const void* x, const void* w, const void* bias, int32_t bias_dtype, const void* y, const void* values, const void* scales) {
    if (!x || !w || !y || !values != !scales) return fail(NDC_ERR_INVALID, "q8 linear: x, w and y must not be NULL, values and scales come together");
    if (bias && bias_dtype != NDC_F32 && bias_dtype != NDC_BF16) return fail(NDC_ERR_INVALID, "q8 linear: bias dtype must be NDC_F32 or NDC_BF16");
    return NDC_OK;
}

int launch_forward(int batch, int ci, int co, long long n, Parts parts, const void* x, const void* w, const void* bias, int32_t bias_dtype, void* y, void* values,
                   void* scales, void* stream) {
    if (((uintptr_t)x | (uintptr_t)w | (uintptr_t)y | (uintptr_t)values) & 15) return fail(NDC_ERR_ALIGNMENT, "q8 linear: x, w, y and values must lie on 16 bytes");
    if (off_elements(bias_dtype, {bias})) return fail(NDC_ERR_ALIGNMENT, "q8 linear: bias misaligned");
    if (ndc::tc::take_expired()) return fail(NDC_ERR_TIMEOUT, "a wait inside a kernel of an earlier call ran out after one second");
    ForwardArgs P{};
    P.bias = bias; P.bias_bf16 = bias_dtype == NDC_BF16; P.values = (unsigned char*)values; P.scales = (unsigned char*)scales;
    P.n = n; P.pitch = pitch_of(n); P.scale_pitch = (int)scales_of(n);
    P.ci = ci; P.co = co; P.blocks = (ci + KC - 1) / KC; P.columns = parts.columns;
    P.tiles_n = (int)((n + MT - 1) / MT); P.tiles = P.tiles_n * batch;
    const int weights = P.blocks * P.columns * 128;
    P.staged = kRoom - weights - 4 * kStaged >= 4 * kBlockBytes ? 2 : 1;
    P.slots = std::min(kMostSlots, (kRoom - weights - 2 * P.staged * kStaged) / kBlockBytes);
    P.buffers = P.columns <= 256 ? 2 : 1;
    cudaError_t e = ndc::tc::expired_word(P.expired);
    if (e != cudaSuccess) return fail(NDC_ERR_CUDA, "q8 linear: %s", cudaGetErrorString(e));
    CUtensorMap map_x, map_w, map_y;
    if (!make_tensor_map(map_x, x, 2, batch, ci, n, KC) || !make_tensor_map(map_y, y, 2, batch, co, n, MT) || !make_weight_map(map_w, w, co, ci)) return fail(NDC_ERR_CUDA, "q8 linear: the driver refused a tensor map");
    const auto kern = parts.parts > 1 ? forward_kernel<true> : forward_kernel<false>;
    e = ndc::allow_smem(kern);
    if (e == cudaSuccess) {
        kern<<<dim3(ctas_of(P.tiles, parts.parts), parts.parts), kThreads,
                         1024 + kHeader + weights + (size_t)2 * P.staged * kStaged + (size_t)P.slots * kBlockBytes, (cudaStream_t)stream>>>(map_x, map_w, map_y, P);
        ndc::launched();
        e = cudaGetLastError();
    }
    return e == cudaSuccess ? NDC_OK : fail(NDC_ERR_CUDA, "q8 linear: %s", cudaGetErrorString(e));
}

}  // namespace
}  // namespace q8
}  // namespace ndc

using namespace ndc::q8;

extern "C" {

int32_t ndc_q8_linear_fwd_applies(int32_t batch, int32_t ci, int32_t co, int64_t n) {
    return ci > 0 && co > 0 && ci % 8 == 0 && co <= 512 && (long long)ci * co <= kMostWeights && weight_bytes(ci, co) <= kMostWeights && fits_positions(batch, n);
}

int ndc_q8_linear_fwd(int32_t batch, int32_t ci, int32_t co, int64_t n, const void* x, const void* w, const void* bias, int32_t bias_dtype, void* y, void* values,
                      void* scales, void* stream) {
    const int st = check_forward(x, w, bias, bias_dtype, y, values, scales);
    if (st != NDC_OK) return st;
    if (!ndc_q8_linear_fwd_applies(batch, ci, co, n)) return fail(NDC_ERR_UNSUPPORTED, "q8 linear: not for %d x %d channels and these positions", ci, co);
    return launch_forward(batch, ci, co, n, Parts{(co + MT - 1) / MT * MT, 1}, x, w, bias, bias_dtype, y, values, scales, stream);
}

int32_t ndc_q8_linear_fwd_parts_applies(int32_t batch, int32_t ci, int32_t co, int64_t n) {
    return ci > 0 && co > 0 && ci % 8 == 0 && ci <= 512 && co <= 1 << 20 && fits_positions(batch, n);
}

int ndc_q8_linear_fwd_parts(int32_t batch, int32_t ci, int32_t co, int64_t n, const void* x, const void* w, const void* bias, int32_t bias_dtype, void* y,
                            void* values, void* scales, void* stream) {
    const int st = check_forward(x, w, bias, bias_dtype, y, values, scales);
    if (st != NDC_OK) return st;
    if (!ndc_q8_linear_fwd_parts_applies(batch, ci, co, n)) return fail(NDC_ERR_UNSUPPORTED, "q8 linear: not for %d x %d channels and these positions", ci, co);
    return launch_forward(batch, ci, co, n, plan_parts(ci, co), x, w, bias, bias_dtype, y, values, scales, stream);
}

}  // extern "C"
