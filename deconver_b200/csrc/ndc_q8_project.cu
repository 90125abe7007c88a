// A 1x1 projection in 8 bits, from a channels-first tensor as it lies:
//
//     y[b, o, p] = sum over c of w[o, c] x[b, c, p] (+ bias[o])
//
// with x held in blocks of 128 channels at each position and w (held before, rows of channels) in blocks of
// 128 channels: what ndc_q8_hold_channels and ndc_q8_product compute, without x's way through memory in between.  A
// persistent CTA takes 128 positions of a sample after another:
//
//   sixteen warps hold x: a group of four (float32: eight) has a block of 128 channels of the tile in registers,
//       finds each position's largest magnitude, and writes the e4m3 rows into shared memory in the swizzle of the MMA's
//       operands, and the powers of two as the MMA's block scales.  The loads of the other groups' blocks are on their
//       way meanwhile: 128 KB per multiprocessor, which is what keeps the memory busy.
//   one fetches w by TMA, one its scales, one issues the MMAs: a tile's blocks (up to four, 512 channels) stay for all
//       outputs, w comes in chunks of 128 outputs x 128 channels through a ring; a w that fits the ring is fetched once.
//   four store the results, of one accumulator in TMEM while the next is being computed.  The rows of the product are the
//       outputs: a thread has neighbouring positions of one, and writes 16 bytes of them at a time into shared memory, from
//       where they go out by TMA, or, where rows are not whole vectors, by all of the warps row by row.  (With positions as
//       rows a warp stored 32 neighbours of a channel, four instructions for each 2 bytes: 293 us for 256 -> 64
//       channels over 128^3 positions when the loads still were of two positions, 267 this way.)
//
// 256 -> 64 channels over 128^3 positions of bfloat16 take 247 us (1342 MB, 5.4 TB/s), bound by the instructions of the holding warps;
// 2 x (64 -> 256) x 64^3 74 us (4.6 TB/s); 16 x (512 -> 2048) x 4096 100 us, 1370 TFLOP/s, by the results' way out and the
// chunks of w from the L2 cache.
#include <algorithm>
#include <type_traits>

#include "ndc_b200.h"
#include "ndc_common.cuh"
#include "ndc_q8_host.h"
#include "ndc_q8_mma.cuh"
#include "ndc_q8_rows.cuh"
#include "ndc_tc_host.h"

namespace ndc {
namespace q8 {
namespace {

typedef __nv_bfloat16 bf16;

constexpr int kHoldWarps = 16, kStoreWarps = 4;
constexpr int kThreads = 32 * (kHoldWarps + kStoreWarps + 3);
constexpr int kMostBlocks = 4;               // of channels
constexpr int kPlaces = 2, kStaged = MT * 128;       // results on their way out: 128 outputs x 128 bytes of positions
constexpr int kOperands = 10;                // blocks of x and of w in shared memory, 16 KB each
constexpr int kSlots = 4;                    // of x: a tile's blocks, and not fewer than groups (a barrier's phases may not lap a group)
static_assert(kSlots >= kMostBlocks && kSlots >= kHoldWarps / 4, "slots");
constexpr int kOperand = MT * KT;

struct ProjectArgs {
    const void* x;
    const unsigned char* sw;                 // w's scales: a word per row
    const void* bias;                        // float32, or bfloat16, or NULL
    int bias_bf16;
    void* y;
    long long n;                             // positions of a sample
    int ci, co, blocks, chunks;              // blocks of input channels, chunks of output channels
    int tiles_n;                             // of a sample
    int parts, items;                        // a tile's chunks are shared by `parts` CTAs; items = tiles * parts
    int resident;                            // w stays in the ring
    int stages;                              // blocks of w in the ring
    Divider by_tiles_n, by_parts, by_blocks;
    unsigned* expired;
};

// Barriers and scales have room for as many of either as there are blocks.
constexpr int kGaveUp = 512, kTops = 1024, kScalesX = kTops + 8192, kScalesW = kScalesX + kOperands * 512, kStaging = (kScalesW + kOperands * 512 + 1023) / 1024 * 1024;
constexpr int kFirst = kStaging + kPlaces * kStaged;
constexpr size_t kSmem = 1024 + kFirst + (size_t)kOperands * kOperand;
static_assert(kSmem <= 227 * 1024, "shared memory");
constexpr int kScaleColumns = 256, kTmem = 512;      // of TMEM: two accumulators, scales

__device__ __forceinline__ void store_sync() { asm volatile("bar.sync 8, 128;" ::: "memory"); }
// Positions h .. h + 31 of a place's row, in its swizzle.
__device__ __forceinline__ void put32(unsigned char* to, int row, int h, const float (&v)[32], bf16*) {
#pragma unroll
    for (int m = 0; m < 4; ++m) {
        unsigned w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 q = __floats2bfloat162_rn(v[8 * m + 2 * i], v[8 * m + 2 * i + 1]);
            w[i] = *reinterpret_cast<const unsigned*>(&q);
        }
        *reinterpret_cast<uint4*>(to + (((h / 8 + m) ^ (row & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}
__device__ __forceinline__ void put32(unsigned char* to, int row, int, const float (&v)[32], float*) {
#pragma unroll
    for (int m = 0; m < 8; ++m) *reinterpret_cast<float4*>(to + ((m ^ (row & 7)) << 4)) = make_float4(v[4 * m], v[4 * m + 1], v[4 * m + 2], v[4 * m + 3]);
}

// TMA: results out by it.
template <typename T, bool VEC, bool TMA>
__global__ void __launch_bounds__(kThreads, 1) project_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_y,
                                                              const __grid_constant__ ProjectArgs P) {
    // (rows whose results go out by TMA are whole vectors, x's whole ones of four)
    constexpr bool QUADS = TMA && sizeof(T) == 2;
    static_assert(VEC || !TMA, "TMA");
    using R = std::conditional_t<QUADS, Quads, Rows<T, VEC>>;
    constexpr int GROUPS = kHoldWarps / R::WARPS;
    static_assert(GROUPS * 16 * MT <= kScalesX - kTops, "groups' largest magnitudes");
    extern __shared__ unsigned char raw_smem[];
    unsigned char* smem = raw_smem + ((1024u - (smem_u32(raw_smem) & 1023u)) & 1023u);
    const unsigned base = smem_u32(smem);
    const unsigned afull = base, aempty = afull + 8 * kOperands, bfull = aempty + 8 * kOperands, bempty = bfull + 8 * kOperands;
    const unsigned dfull = bempty + 8 * kOperands, dempty = dfull + 16, slot_at = dempty + 16;
    // a group of warps whose wait ran out, as seen by all of it after their next barrier: they leave it together
    volatile unsigned* const gave_up = reinterpret_cast<volatile unsigned*>(smem + kGaveUp);
    const unsigned x_at = base + kFirst, w_at = x_at + kSlots * kOperand;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < kSlots; ++i) { mbar_init(afull + 8 * i, R::WARPS); mbar_init(aempty + 8 * i, 1); }
        for (int i = 0; i < P.stages; ++i) { mbar_init(bfull + 8 * i, 2); mbar_init(bempty + 8 * i, 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(dfull + 8 * i, 1); mbar_init(dempty + 8 * i, kStoreWarps); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (threadIdx.x <= GROUPS) gave_up[threadIdx.x] = 0u;      // the last one: the storing warps
    if (warp == kHoldWarps) tmem_alloc(slot_at, kTmem);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const unsigned tmem = *reinterpret_cast<volatile unsigned*>(smem + (slot_at - base));
    const int KB = P.blocks;
    bool ok = true;
    // the chunks of an item
    auto first_chunk = [&](int item) { return P.parts == 1 ? 0 : (int)P.by_parts.quotient((unsigned)P.chunks * P.by_parts.remainder((unsigned)item)); };
    auto last_chunk = [&](int item) { return P.parts == 1 ? P.chunks : (int)P.by_parts.quotient((unsigned)P.chunks * (P.by_parts.remainder((unsigned)item) + 1u)); };
    struct Place { int sample; unsigned first; };          // of an item's tile
    auto place_of = [&](int item) {
        const unsigned tile = P.by_parts.quotient((unsigned)item), sample = P.by_tiles_n.quotient(tile);
        return Place{(int)sample, (tile - sample * (unsigned)P.tiles_n) * MT};
    };

    if (warp < kHoldWarps) {
        const int group = warp / R::WARPS, w = warp % R::WARPS, row = R::position(w, lane), share = R::share(w);
        unsigned* tops = reinterpret_cast<unsigned*>(smem + kTops) + group * (4 * MT);     // [2][share][positions]
        int turn = 0;
        for (int q = group;; q += GROUPS, turn ^= 1) {
            const int mine = (int)P.by_blocks.quotient((unsigned)q), kb = q - mine * KB, item = blockIdx.x + mine * gridDim.x;
            if (item >= P.items) break;
            const int c0 = kb * KT + R::CHANNELS * share, channels = min(R::CHANNELS, P.ci - c0);
            const Place at = place_of(item);
            // positions past the last one are computed from it (pairs: the last one), and not stored
            const unsigned n = (unsigned)P.n, i = at.first + row, last = n - (VEC ? R::PER : 1);
            unsigned r[64], top[R::PER];
            R::load(reinterpret_cast<const T*>(P.x) + ((long long)at.sample * P.ci + c0) * P.n, min(i, last), min(i + 1, last), n, channels, r);
            bool told;
            if constexpr (QUADS) told = tops_of_quads(r, top, group, share, tops + turn * (2 * MT), lane, !ok);
            else told = tops_of<R>(r, top, group, share, tops + turn * (2 * MT) + row, !ok);
            if (told && gave_up[group]) break;
            const int use = q / kSlots, s = q % kSlots;
            if (use && !mbar_wait(aempty + 8 * s, (use - 1) & 1)) {
                ok = false;
                gave_up[group] = 1u;
                continue;
            }
#pragma unroll
            for (int i = 0; i < R::PER; ++i) {
                const unsigned byte = scale_byte(top[i]);
                const unsigned long long inv = both(scale_inverse(byte));
                const int at = row + i;
                unsigned char* to = smem + kFirst + s * kOperand + at * KT;
#pragma unroll
                for (int m = 0; m < R::CHANNELS / 16; ++m)
                    if (16 * m < ((channels + 31) & ~31))        // no MMA reads further
                        *reinterpret_cast<uint4*>(to + (((R::CHANNELS / 16 * share + m) ^ (at & 7)) << 4)) = encode16<R>(r, 16 * m, i, inv);
                if (share == 0) smem[kScalesX + s * 512 + (at & 31) * 16 + (at >> 5) * 4] = (unsigned char)byte;
            }
            fence_async_proxy();
            __syncwarp();
            if (lane == 0) mbar_arrive(afull + 8 * s);
        }
    } else if (warp < kHoldWarps + kStoreWarps) {
        constexpr int E = 128 / (int)sizeof(T);              // positions of a place
        const int w = warp - kHoldWarps, row = 32 * w + lane;
        const bool copies = TMA && row == 0;
        int count = 0, place = 0;
        for (int item = blockIdx.x; item < P.items && ok; item += gridDim.x) {
            const Place at = place_of(item);
            const int end = last_chunk(item);
            for (int c = first_chunk(item); c < end && ok; ++c, ++count) {
                const int d = count & 1, o0 = c * MT, outputs = min(MT, P.co - o0);
                const float bias = P.bias && row < outputs ? load_bias(P.bias, P.bias_bf16, o0 + row) : 0.0f;
                if (!mbar_wait(dfull + 8 * d, (count >> 1) & 1)) { ok = false; gave_up[GROUPS] = 1u; }
                tc_fence_after();
#pragma unroll 1
                for (int p0 = 0; p0 < MT; p0 += E, place ^= 1) {
                    unsigned char* to = smem + kStaging + place * kStaged;
                    if (copies) copies_read<1>();            // the place is free where its last copy has read it
                    store_sync();
                    if (gave_up[GROUPS]) { ok = false; break; }
#pragma unroll
                    for (int h = 0; h < E; h += 32) {
                        if (32 * w >= outputs) break;        // nothing of it goes out
                        float v[32];
                        tmem_load32(tmem + ((unsigned)(32 * w) << 16) + d * MT + p0 + h, v);
#pragma unroll
                        for (int j = 0; j < 32; ++j) v[j] += bias;
                        put32(to + row * 128, row, h, v, reinterpret_cast<T*>(to));
                    }
                    if (p0 + E >= MT) {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(dempty + 8 * d);
                    }
                    if (TMA) {
                        fence_async_proxy();
                        store_sync();
                        if (copies) tma_store3(&map_y, at.first + p0, o0, at.sample, base + kStaging + place * kStaged, at.first + p0 < (unsigned)P.n);
                    } else {
                        store_sync();
                        // a row's neighbours by a warp; eight rows are read before the first one is stored
                        const unsigned n = (unsigned)P.n, left = at.first + p0 < n ? n - at.first - p0 : 0;
                        const long long step = kStoreWarps * P.n;
#pragma unroll
                        for (int j = 0; j < E; j += 32) {
                            T* y = reinterpret_cast<T*>(P.y) + ((long long)at.sample * P.co + o0 + w) * P.n + at.first + p0 + j + lane;
                            // (rows w and w + 4 are in turn where the swizzle has them)
                            constexpr int S = (int)sizeof(T);
                            const int in = (j + lane) * S, even = w * 128 + (((in >> 4) ^ w) << 4) + (in & 15), odd = (w + 4) * 128 + (((in >> 4) ^ (w + 4)) << 4) + (in & 15);
                            for (int o = w; o < outputs; o += 8 * kStoreWarps) {
                                T f[8];
#pragma unroll
                                for (int k = 0; k < 8; ++k) f[k] = *reinterpret_cast<const T*>(to + (o - w) * 128 + (k & 1 ? odd : even) + k / 2 * 1024);
#pragma unroll
                                for (int k = 0; k < 8; ++k, y += step)
                                    if (o + kStoreWarps * k < outputs && j + lane < left) *y = f[k];
                            }
                        }
                    }
                }
            }
        }
        if (copies) copies_done();
    } else if (warp == kHoldWarps + kStoreWarps) {
        if (lane == 0) {
            int count = 0;                       // of the stages that were filled
            auto fetch = [&](int c, int kb) {
                const int use = count / P.stages, s = count - use * P.stages;
                if (use) ok = mbar_wait_thread(bempty + 8 * s, (use - 1) & 1, kWaitLimit);
                if (!ok) return;
                expect_bytes(bfull + 8 * s, kOperand);
                tma_load(w_at + s * kOperand, &map_w, kb * KT, c * MT, bfull + 8 * s);
                ++count;
            };
            for (int item = blockIdx.x; item < P.items && ok; item += gridDim.x) {
                const int end = last_chunk(item);
                for (int c = first_chunk(item); c < end && ok; ++c)
                    for (int kb = 0; kb < KB && ok; ++kb) fetch(c, kb);
                if (P.resident) break;
            }
            // copies that nobody may have waited for
            for (int t = max(0, count - P.stages); t < count; ++t) mbar_wait_thread(bfull + 8 * (t % P.stages), (t / P.stages) & 1, kWaitLimit);
        }
    } else if (warp == kHoldWarps + kStoreWarps + 1) {
        int count = 0;
        for (int item = blockIdx.x; item < P.items && ok; item += gridDim.x) {
            const int end = last_chunk(item);
            for (int c = first_chunk(item); c < end && ok; ++c) {
                unsigned u[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) u[i] = __ldg(reinterpret_cast<const unsigned*>(P.sw) + min(P.co - 1, c * MT + 32 * i + lane));
                for (int kb = 0; kb < KB; ++kb, ++count) {
                    const int use = count / P.stages, s = count - use * P.stages;
                    if (use) ok = mbar_wait(bempty + 8 * s, (use - 1) & 1);
                    if (!ok) break;
                    *reinterpret_cast<uint4*>(smem + kScalesW + s * 512 + 16 * lane) = make_uint4(u[0], u[1], u[2], u[3]);
                    fence_async_proxy();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bfull + 8 * s);
                }
            }
            if (P.resident) break;
        }
    } else {
        if (elect()) {
            // the next stage of w and slot of x, and the phases of their barriers
            int chunk = 0, st = 0, sphase = 0, x0 = 0, xphase = 0;
            bool fresh = true;
            for (int item = blockIdx.x; item < P.items && ok; item += gridDim.x) {
                const int begin = first_chunk(item), end = last_chunk(item);
                for (int c = begin; c < end && ok; ++c, ++chunk) {
                    const int d = chunk & 1;
                    if (chunk >= 2) ok = mbar_wait_thread(dempty + 8 * d, ((chunk >> 1) - 1) & 1, kWaitLimit);
                    if (!ok) break;
                    int sx = x0, phase = xphase;
                    for (int kb = 0; kb < KB; ++kb) {
                        const unsigned sfx = tmem + kScaleColumns + 4 * sx, sfw = tmem + kScaleColumns + 4 * (kSlots + st);
                        if (c == begin) ok = mbar_wait_thread(afull + 8 * sx, phase, kWaitLimit);
                        if (ok && fresh) ok = mbar_wait_thread(bfull + 8 * st, sphase, kWaitLimit);
                        if (!ok) break;
                        tc_fence_after();
                        const unsigned long long x = swizzled_desc(x_at + sx * kOperand), w = swizzled_desc(w_at + st * kOperand);
                        const unsigned idesc = scaled_instr(MT, kb, 0);
                        const int steps = (P.ci - kb * KT + 31) / 32;
                        {
                            if (c == begin) scales_to_tmem(sfx, mat_desc(base + kScalesX + sx * 512, 128, 128));
                            if (fresh) scales_to_tmem(sfw, mat_desc(base + kScalesW + st * 512, 128, 128));
#pragma unroll
                            for (int i = 0; i < KT / 32; ++i)
                                if (i < steps) mma_scaled(tmem + d * MT, w + 2 * i, x + 2 * i, idesc, sfw, sfx, kb > 0 || i > 0);
                            if (!P.resident) mma_commit(bempty + 8 * st);
                            if (c == end - 1) mma_commit(aempty + 8 * sx);
                            if (kb == KB - 1) mma_commit(dfull + 8 * d);
                        }
                        if (++sx == kSlots) { sx = 0; phase ^= 1; }
                        if (++st == P.stages) { st = 0; sphase ^= 1; }
                    }
                    if (c == end - 1) { x0 = sx; xphase = phase; }
                }
                if (P.resident) { fresh = false; st = 0; }
            }
        }
    }
    if (!ok) report_expired(P.expired);
    __syncwarp();
    __syncthreads();
    if (warp == kHoldWarps) {
        tc_fence_after();
        tmem_free(tmem, kTmem);
    }
}

// CTAs that share a tile's chunks of outputs, each holding the tile's x: the least rounds of CTAs times chunks, where x counts as 2.4
// (16 x (512 -> 2048) channels x 4096 positions, 512 tiles of 16 chunks: by one 108 us, by two 100; 3 x (512 -> 512) x 8000 27 and 29).  A w that
// stays is not shared where there are tiles for all.
int plan_parts(long long tiles, int chunks, int blocks) {
    const long long sms = ndc::num_sms();
    int best = 1;
    double best_time = 1e300;
    for (int parts = 1; parts <= std::min(chunks, (int)sms); ++parts) {
        if (parts > 1 && chunks * blocks <= kMostBlocks && tiles >= sms) break;
        const double time = (double)((tiles * parts + sms - 1) / sms) * ((chunks + parts - 1) / parts + 2.4);
        if (time < best_time) { best_time = time; best = parts; }
    }
    return best;
}

template <typename T, bool VEC, bool TMA>
cudaError_t launch(const CUtensorMap& map_w, const CUtensorMap& map_y, const ProjectArgs& P, cudaStream_t st) {
    auto kern = project_kernel<T, VEC, TMA>;
    const cudaError_t e = ndc::allow_smem(kern);
    if (e != cudaSuccess) return e;
    kern<<<(unsigned)std::min(P.items, ndc::num_sms()), kThreads, 1024 + kFirst + (size_t)(kSlots + P.stages) * kOperand, st>>>(map_w, map_y, P);
    ndc::launched();
    return cudaGetLastError();
}

}  // namespace
}  // namespace q8
}  // namespace ndc

using namespace ndc::q8;

extern "C" {

int ndc_q8_project(int32_t batch, int32_t ci, int32_t co, int64_t n, int32_t dtype, const void* x, const void* w_values, const void* w_scales,
                   const void* bias, int32_t bias_dtype, void* y, void* stream) {
    if (!x || !w_values || !w_scales || !y) return fail(NDC_ERR_INVALID, "q8 projection: x, w and y must not be NULL");
    if (batch <= 0 || ci <= 0 || co <= 0 || n <= 0) return fail(NDC_ERR_INVALID, "q8 projection: extents must be positive");
    if ((dtype != NDC_F32 && dtype != NDC_BF16) || (bias && bias_dtype != NDC_F32 && bias_dtype != NDC_BF16)) return fail(NDC_ERR_INVALID, "q8 projection: dtype must be NDC_F32 or NDC_BF16");
    const int blocks = (ci + kBlock - 1) / kBlock;
    const long long tiles_n = (n + MT - 1) / MT, tiles = batch * tiles_n;
    // (chunks times parts stay below 2^31)
    if (blocks > kMostBlocks || n > kMostPositions || co > 1 << 30 || tiles > (0x7fffffffLL - 65536) / ((co + MT - 1) / MT))
        return fail(NDC_ERR_UNSUPPORTED, "q8 projection: more than %d channels, or too many positions or outputs", kMostBlocks * kBlock);
    if ((uintptr_t)w_values & 15 || (uintptr_t)w_scales & 3) return fail(NDC_ERR_ALIGNMENT, "q8 projection: values on 16 bytes, scales on 4");
    if (off_elements(dtype, {x, y}) || off_elements(bias_dtype, {bias})) return fail(NDC_ERR_ALIGNMENT, "q8 projection: a tensor does not lie on its elements' size");
    if (ndc::tc::take_expired()) return fail(NDC_ERR_TIMEOUT, "a wait inside a kernel of an earlier call ran out after one second");
    const int parts = plan_parts(tiles, (co + MT - 1) / MT, blocks);
    ProjectArgs P{x, (const unsigned char*)w_scales, bias, bias_dtype == NDC_BF16, y, n, ci, co, blocks, (co + MT - 1) / MT, (int)tiles_n, parts, (int)(tiles * parts),
                  0, 0, Divider((unsigned)tiles_n), Divider((unsigned)parts), Divider((unsigned)blocks), nullptr};
    // A w of up to four blocks stays.  One that goes around needs many on their way, and the tile's blocks change seldom.
    P.resident = P.parts == 1 && P.chunks * blocks <= kMostBlocks;
    P.stages = P.resident ? P.chunks * blocks : kOperands - kSlots;
    cudaError_t e = ndc::tc::expired_word(P.expired);
    if (e != cudaSuccess) return fail(NDC_ERR_CUDA, "q8 projection: %s", cudaGetErrorString(e));
    const int size = dtype == NDC_F32 ? 4 : 2;
    const bool tma = n * size % 16 == 0 && ((uintptr_t)y & 15) == 0 && ((uintptr_t)x & (size == 4 ? 3 : 7)) == 0, vec = dtype == NDC_F32 || (n % 2 == 0 && ((uintptr_t)x & 3) == 0);
    CUtensorMap map_w, map_y{};
    if (!make_map(map_w, w_values, co, pitch_of(ci), MT) || (tma && !make_tensor_map(map_y, y, size, batch, co, n, MT)))
        return fail(NDC_ERR_CUDA, "q8 projection: the driver refused a tensor map");
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == NDC_F32) e = tma ? launch<float, true, true>(map_w, map_y, P, st) : launch<float, true, false>(map_w, map_y, P, st);
    else if (tma) e = launch<bf16, true, true>(map_w, map_y, P, st);
    else e = vec ? launch<bf16, true, false>(map_w, map_y, P, st) : launch<bf16, false, false>(map_w, map_y, P, st);
    return e == cudaSuccess ? NDC_OK : fail(NDC_ERR_CUDA, "q8 projection: %s", cudaGetErrorString(e));
}

}  // extern "C"
