// The weight gradient of a 1x1 projection from the held input (format: ndc_q8.cuh), and the bias gradient:
//
//     gw[o, c] = sum over samples and positions of gy[b, o, p] v[b, c, p],      gb[o] = sum of gy[b, o, p]
//
// for what is held, v.  Every held value is a bfloat16 value (four significant bits and a power of two), so the
// products are those of bfloat16 operands, exact in float32, and summed in float32 on the tensor cores.  float32
// gradients go as three bfloat16 terms of eight bits each, which together are the value: three products instead of the six
// of two split operands.  The MMA cuts its sums off towards zero, by up to 2^-23 of them each time, so that a chain of m shrinks by
// m 2^-25 to m 2^-24 (values of one sign): sums go into several accumulators in turn (as many as TMEM has room for), float32's small terms' into one of
// their own, and a slice is no longer than kChain or kChain16 in each (float32, 2 x (11 -> 63) channels x 80000 positions: 1.5e-5 of the result in
// one chain; bfloat16, (256 -> 1000) x 2^20: 4.3e-4, where the rounding of the result is 2^-9 of it on the average).  Slices whose sums would
// be too much memory go in several launches (plan_passes).  The bias gradient comes from sixteen more columns of the product, of rows of ones; one
// that is not finite is added up by itself.
// 2 x (64 -> 256) x 64^3 in bfloat16: 62 us and 4 for the slices' sums (303 MB, 4.9 TB/s), bound by memory and by the held rows' way
// through registers; 5 x (24 -> 96) of 203x171 in float32: 40 us, by loads of gy one value at a time and their split.
//
// A CTA has a tile of 128 outputs x up to 240 inputs and a slice of the positions, 64 at a time in a ring of stages in
// shared memory (K-major, 128-byte swizzle).  bfloat16 gradients in rows of whole vectors come by TMA, and sixteen warps, in
// two groups that take turns, bring the held rows as bfloat16; else they bring both.  (All
// warps at every step with two steps' loads on their way in registers waited for both at the first one's use: 129 us at 2 x (256 +
// 64) x 64^3, a third of the memory's rate.)  One warp issues the MMAs; the slices' sums are added by a second kernel in a
// fixed order, which converts to the parameters' types.
#include <algorithm>
#include <type_traits>

#include "ndc_b200.h"
#include "ndc_common.cuh"
#include "ndc_q8_host.h"
#include "ndc_q8_mma.cuh"
#include "ndc_tc_host.h"

namespace ndc {
namespace q8 {
namespace {

typedef __nv_bfloat16 bf16;

constexpr int kStageWarps = 16, kStagers = 32 * kStageWarps, kThreads = kStagers + 64;     // two for the MMAs and TMA
constexpr int KP = 64;                        // positions of a row of 128 bytes of bfloat16
constexpr int kRowBytes = 2 * KP;
constexpr int kMostColumns = 256;             // of a tile, with the ones' 16
constexpr int kTmem = 512;
constexpr int kChain = 64;                    // MMAs of float32's leading terms into one accumulator
constexpr int kChain16 = 1024;                // of bfloat16's: 2^-14 of a sum at most (2^-18 of a bias gradient's, of sixteen rows), rounded to 2^-8
constexpr int kHeader = 1024;

struct WgradArgs {
    const void* gy;
    const unsigned char *values, *scales;
    float* partial;                           // [slice][width][co]: a warp's lanes have neighbouring outputs
    long long n, pitch;
    int scale_pitch;
    int co, ci, ct, width;                    // inputs of a tile (a multiple of 16); ci, and one more with a bias
    int steps_n;                              // steps of a sample
    long long steps;                          // of all samples
    int slices, slice0;                       // of all; the launch's first one
    unsigned* expired;
};

// A step has SUB times 64 positions: two where they come by TMA (rows' 256 bytes at once: 128 left the memory at two thirds of its
// rate), one where float32's three terms take the room.
template <typename T, bool VEC> struct Step {
    static constexpr bool TMA = VEC && sizeof(T) == 2;
    static constexpr int TERMS = sizeof(T) == 4 ? 3 : 1, SUB = TMA ? 2 : 1, POSITIONS = SUB * KP;
    static constexpr int G = TERMS * MT * kRowBytes;      // bytes of 64 positions of gy
    __host__ __device__ static constexpr int bytes(int columns) { return SUB * (G + columns * kRowBytes); }
};
// columns of a tile's product
__host__ __device__ inline int columns_of(int ct) { return ct + 16; }
// Accumulators that sums go into in turn: what TMEM has room for (float32: beside that of the small terms), whole 32 columns read past their end.
__host__ __device__ inline int leading_of(int columns, int terms) {
    const int n = (kTmem - 16) / columns - (terms > 1 ? 1 : 0);
    return n < 1 ? 1 : n > 15 ? 15 : n;
}
template <typename S> int stages_of(int ct) { return std::min(6, (int)((227 * 1024 - 1024 - kHeader) / S::bytes(columns_of(ct)))); }

// Eight positions of a row of gy; zeros past its end.
template <typename T, bool VEC> struct Octet;
template <bool VEC> struct Octet<bf16, VEC> {
    uint4 q;
    __device__ __forceinline__ void load(const bf16* p, long long left) {
        if (VEC) {
            q = left > 0 ? __ldg(reinterpret_cast<const uint4*>(p)) : make_uint4(0u, 0u, 0u, 0u);
        } else {
            const unsigned short* u = reinterpret_cast<const unsigned short*>(p);
            unsigned w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = i < left ? __ldg(u + i) : 0u;
            q = make_uint4(w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16);
        }
    }
    __device__ __forceinline__ void store(unsigned char* to) const { *reinterpret_cast<uint4*>(to) = q; }
};
template <bool VEC> struct Octet<float, VEC> {
    float v[8];
    __device__ __forceinline__ void load(const float* p, long long left) {
        if (VEC) {
#pragma unroll
            for (int i = 0; i < 8; i += 4) {
                const float4 f = i < left ? __ldg(reinterpret_cast<const float4*>(p + i)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                v[i] = f.x; v[i + 1] = f.y; v[i + 2] = f.z; v[i + 3] = f.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = i < left ? __ldg(p + i) : 0.0f;
        }
    }
    // the leading eight bits of each value, the next eight, and the last; an infinity has no remainder (a NaN does: it may have its bits below the leading ones)
    __device__ __forceinline__ void store(unsigned char* to) {
#pragma unroll
        for (int t = 0; t < 3; ++t) {
            unsigned w[4];
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                const unsigned a = __float_as_uint(v[i]), b = __float_as_uint(v[i + 1]);
                w[i / 2] = __byte_perm(a, b, 0x7632);
                if (t < 2) {
                    const unsigned ha = a & 0xffff0000u, hb = b & 0xffff0000u;
                    v[i] = (a & 0x7fffffffu) == kInfinite ? 0.0f : v[i] - __uint_as_float(ha);
                    v[i + 1] = (b & 0x7fffffffu) == kInfinite ? 0.0f : v[i + 1] - __uint_as_float(hb);
                }
            }
            *reinterpret_cast<uint4*>(to + t * MT * kRowBytes) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
};

__device__ __forceinline__ unsigned decode_bf16(unsigned pair, float scale) {
    const float2 f = decode2(pair);
    const __nv_bfloat162 p = __floats2bfloat162_rn(f.x * scale, f.y * scale);
    return *reinterpret_cast<const unsigned*>(&p);
}

// The sum of a row of gy over some steps, by a warp; no further than to what makes it NaN.
template <typename T>
__device__ __forceinline__ float row_sum(const WgradArgs& P, int o, long long first, int steps, int positions, int lane) {
    float s = 0.0f;
    for (long long step = first; step < first + steps; ++step) {
        const long long sample = step / P.steps_n, p = (step - sample * P.steps_n) * positions, left = min((long long)positions, P.n - p);
        const T* g = reinterpret_cast<const T*>(P.gy) + (sample * P.co + o) * P.n + p;
        for (int i = lane; i < left; i += 32) s += ndc::to_f32(g[i]);
        const float inf = __uint_as_float(kInfinite);
        if (__any_sync(0xffffffffu, s != s) || (__any_sync(0xffffffffu, s == inf) && __any_sync(0xffffffffu, s == -inf))) return __uint_as_float(0x7fffffffu);
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    return s;
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads, 1) wgrad_kernel(const __grid_constant__ CUtensorMap map_g, const __grid_constant__ WgradArgs P, int stages) {
    typedef Step<T, VEC> S;
    constexpr bool TMA = S::TMA;
    constexpr int GROUPS = 2, WARPS = kStageWarps / GROUPS;
    extern __shared__ unsigned char raw_smem[];
    unsigned char* smem = raw_smem + ((1024u - (smem_u32(raw_smem) & 1023u)) & 1023u);
    const unsigned base = smem_u32(smem);
    const unsigned full = base, empty = base + 64, done = base + 128, slot_at = base + 136;      // up to eight stages
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tid = threadIdx.x;
    const int o0 = blockIdx.x * MT, c0 = blockIdx.y * P.ct;
    const int inputs = min(P.ct, P.ci - c0), columns = columns_of(P.ct), bytes = S::bytes(columns);
    const long long slice = P.slice0 + (int)blockIdx.z, first = P.steps * slice / P.slices;
    const int steps = (int)(P.steps * (slice + 1) / P.slices - first);
    constexpr int B = S::SUB * S::G;                      // where a stage's held rows begin

    if (tid == 0) {
        for (int i = 0; i < stages; ++i) { mbar_init(full + 8 * i, WARPS + (TMA ? 1 : 0)); mbar_init(empty + 8 * i, 1); }
        mbar_init(done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kStageWarps) tmem_alloc(slot_at, kTmem);
    // the ones, in sixteen rows after the tile's inputs; what is not written below is zero.  Each 16 positions of a stage have
    // theirs in another row: the MMA cuts its sums off, so that chains of a sixteenth of the length lose a sixteenth (bias
    // gradient in float32, 2 x 64^3 positions: 3e-6 of it with one row)
    const int extra = columns - inputs;
    for (int i = tid; i < stages * S::SUB * extra * 8; i += kThreads) {
        const int tile = i / (extra * 8), row = inputs + i / 8 % extra, piece = i & 7;       // 16 bytes: eight positions
        const int one = row >= P.ct && (tile * 4 + piece / 2) % 16 == row - P.ct ? 0x3f803f80 : 0;
        unsigned char* to = smem + kHeader + tile / S::SUB * bytes + B + (tile % S::SUB * columns + row) * kRowBytes;
        *reinterpret_cast<int4*>(to + ((piece ^ (row & 7)) << 4)) = make_int4(one, one, one, one);
    }
    fence_async_proxy();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const unsigned tmem = *reinterpret_cast<volatile unsigned*>(smem + (slot_at - base));
    bool ok = true;

    if (warp < kStageWarps) {
        constexpr int ROWS = 4 * WARPS / S::SUB, GU = TMA ? 0 : MT / ROWS, XU = 4;     // units of eight positions per thread, XU held ones at a time
        const int group = warp / WARPS, own = tid % (32 * WARPS), j = own & 7, sub = own / 8 % S::SUB, row = own / 8 / S::SUB;       // of the first; the others are ROWS further on each
        const int swizzled = row * kRowBytes + ((j ^ (row & 7)) << 4);
        for (int t = group; t < steps && ok; t += GROUPS) {
            const long long step = first + t;
            const int sample = (int)(step / P.steps_n);
            const long long p = (step - (long long)sample * P.steps_n) * S::POSITIONS + KP * sub + 8 * j;
            Octet<T, VEC> g[GU + 1];
#pragma unroll
            for (int i = 0; i < GU; ++i) {
                const int o = o0 + row + ROWS * i;
                g[i].load(reinterpret_cast<const T*>(P.gy) + ((long long)sample * P.co + o) * P.n + p, o < P.co ? P.n - p : 0);
            }
            const long long held_row = (long long)sample * P.ci + c0 + row;
            const unsigned char *values = P.values + held_row * P.pitch + p, *scales = P.scales + held_row * P.scale_pitch + p / kBlock;
            const int rows = p < P.pitch ? inputs - row : 0;     // that there are
            uint2 x[XU];
            unsigned char scale[XU];
            auto fetch = [&](int at) {
#pragma unroll
                for (int i = 0; i < XU; ++i) {
                    const bool in = at + ROWS * i < rows;
                    x[i] = in ? __ldg(reinterpret_cast<const uint2*>(values + (at + ROWS * i) * P.pitch)) : make_uint2(0u, 0u);
                    scale[i] = in ? __ldg(scales + (long long)(at + ROWS * i) * P.scale_pitch) : 1;
                }
            };
            fetch(0);
            const int s = t % stages;
            if (t >= stages) ok = mbar_wait(empty + 8 * s, (t / stages - 1) & 1);
            if (!ok) break;
            unsigned char* to = smem + kHeader + s * bytes + swizzled;
#pragma unroll
            for (int i = 0; i < GU; ++i) g[i].store(to + ROWS * i * kRowBytes);       // (not by TMA: SUB is one)
            to += B + sub * columns * kRowBytes;
            for (int at = 0; at < inputs; at += XU * ROWS) {
                uint4 v[XU];
#pragma unroll
                for (int i = 0; i < XU; ++i) {
                    const float f = scale_value(scale[i]);
                    v[i] = make_uint4(decode_bf16(x[i].x & 0xffffu, f), decode_bf16(x[i].x >> 16, f), decode_bf16(x[i].y & 0xffffu, f), decode_bf16(x[i].y >> 16, f));
                }
                if (at + XU * ROWS < inputs) fetch(at + XU * ROWS);
#pragma unroll
                for (int i = 0; i < XU; ++i)
                    if (at + ROWS * i < inputs - row) *reinterpret_cast<uint4*>(to + (at + ROWS * i) * kRowBytes) = v[i];
            }
            fence_async_proxy();
            __syncwarp();
            if (lane == 0) mbar_arrive(full + 8 * s);
        }
        // four warps for each 32 columns; no branch between a thread's stores (by four warps alone, with a branch each: 21 us for
        // 2 x (512 -> 2048) channels x 512 positions, 14 by all with the branches, 11 without)
        if (ok) ok = mbar_wait(done, 0);
        tc_fence_after();
        const int quarter = warp & 3, o = o0 + 32 * quarter + lane;
        float* out = P.partial + (long long)blockIdx.z * P.width * P.co + o;
        // float32's small terms, then the accumulators of every step in turn
        const int sums = (S::TERMS > 1 ? 1 : 0) + min(steps, leading_of(columns, S::TERMS));
#pragma unroll 1
        for (int k = 32 * (warp >> 2); k < columns; k += 8 * kStageWarps) {
            float v[32];
            __syncwarp();
            tmem_load32(tmem + ((unsigned)(32 * quarter) << 16) + k, v);       // (columns past the last one are not used)
            for (int i = 1; i < sums; ++i) {
                float more[32];
                __syncwarp();
                tmem_load32(tmem + ((unsigned)(32 * quarter) << 16) + i * columns + k, more);
#pragma unroll
                for (int j = 0; j < 32; ++j) v[j] += more[j];
            }
            store_columns(out + (long long)(c0 + k) * P.co, P.co, v, inputs - k, o < P.co && ok, 0.0f, false);
            // the ones' sixteen columns, the first or the last ones of 32
            if (blockIdx.y == 0 && P.width > P.ci && (k == P.ct || k + 16 == P.ct)) {
                float ones = 0.0f;
#pragma unroll
                for (int i = 0; i < 16; ++i) ones += k == P.ct ? v[i] : v[16 + i];
                // An infinity times the other rows' zeros is NaN, whatever the sum is: it is made again, without them
                unsigned odd = __ballot_sync(0xffffffffu, o < P.co && ok && !(fabsf(ones) < __uint_as_float(kInfinite)));
                for (; odd; odd &= odd - 1) {
                    const int l = __ffs(odd) - 1;
                    const float sum = row_sum<T>(P, o0 + 32 * quarter + l, first, steps, S::POSITIONS, lane);
                    if (lane == l) ones = sum;
                }
                if (o < P.co && ok) out[(long long)P.ci * P.co] = ones;
            }
        }
        tc_fence_before();
    } else if (TMA && warp == kStageWarps + 1) {
        if (lane == 0) {
            int t = 0;
            for (; t < steps; ++t) {
                const int s = t % stages;
                if (t >= stages) ok = mbar_wait_thread(empty + 8 * s, (t / stages - 1) & 1, kWaitLimit);
                if (!ok) break;
                const long long step = first + t;
                const int sample = (int)(step / P.steps_n), p = (int)(step - (long long)sample * P.steps_n) * S::POSITIONS;
                expect_bytes(full + 8 * s, S::SUB * S::G);
#pragma unroll
                for (int i = 0; i < S::SUB; ++i) tma_load(base + kHeader + s * bytes + i * S::G, &map_g, p + KP * i, sample * P.co + o0, full + 8 * s);
            }
            if (!ok)               // the copies that are on their way
                for (int i = max(0, t - stages); i < t; ++i) mbar_wait_thread(full + 8 * (i % stages), (i / stages) & 1, kWaitLimit);
        }
    } else if (warp == kStageWarps) {
        if (elect()) {
            const unsigned idesc = instr_desc(columns);
            const int leading = leading_of(columns, S::TERMS), lead0 = S::TERMS > 1 ? columns : 0;
            int lead = lead0;                                               // first column of the step's accumulator
            for (int t = 0; t < steps; ++t) {
                const int s = t % stages;
                ok = mbar_wait_thread(full + 8 * s, (t / stages) & 1, kWaitLimit);
                if (!ok) break;
                tc_fence_after();
                const unsigned at = base + kHeader + s * bytes;
                const unsigned long long g0 = swizzled_desc(at), x0 = swizzled_desc(at + B);
                {
#pragma unroll
                    for (int sub = 0; sub < S::SUB; ++sub) {
                        const unsigned long long x = x0 + sub * columns * (kRowBytes / 16);
#pragma unroll
                        for (int term = S::TERMS - 1; term >= 0; --term)             // the small ones first
#pragma unroll
                            for (int i = 0; i < KP / 16; ++i) {
                            const bool small = S::TERMS > 1 && term > 0;
                            const unsigned to = tmem + (small ? 0 : lead);
                            const bool begun = small ? t > 0 || i > 0 || term < S::TERMS - 1 : t >= leading || sub > 0 || i > 0;
                            mma(to, g0 + (sub * S::G + term * MT * kRowBytes) / 16 + 2 * i, x + 2 * i, idesc, begun);
                        }
                    }
                    lead = lead == lead0 + (leading - 1) * columns ? lead0 : lead + columns;
                    mma_commit(empty + 8 * s);
                }
            }
            mma_commit(done);
        }
    }
    if (!ok) report_expired(P.expired);
    __syncwarp();
    __syncthreads();
    if (warp == kStageWarps) {
        tc_fence_after();
        tmem_free(tmem, kTmem);
    }
}

// gw and gb from the slices' sums: a warp's 32 elements are summed by eight warps, an eighth of the slices each.
template <typename T, typename TB>
__global__ void __launch_bounds__(256) wgrad_sum_kernel(const float* __restrict__ partial, int slices, int co, int ci, int width, T* __restrict__ gw,
                                                        TB* __restrict__ gb) {
    __shared__ float part[8][32];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const long long n = (long long)co * width, e = (long long)blockIdx.x * 32 + lane;
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (e < n) {
        int i = w;
        for (; i + 24 < slices; i += 32)
#pragma unroll
            for (int k = 0; k < 4; ++k) s[k] += partial[(i + 8 * k) * n + e];
        for (; i < slices; i += 8) s[0] += partial[i * n + e];
    }
    part[w][lane] = (s[0] + s[1]) + (s[2] + s[3]);
    __syncthreads();
    if (w == 0 && e < n) {
        float r = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; ++k) r += part[k][lane];
        const long long c = e / co, o = e - c * co;
        if (c < ci) gw[o * ci + c] = ndc::from_f32<T>(r);
        else gb[o] = ndc::from_f32<TB>(r);
    }
}

// The same where there are few slices and many elements: tiles of 32 x 32, read along the outputs and written along the inputs.
template <typename T, typename TB>
__global__ void __launch_bounds__(256) wgrad_few_kernel(const float* __restrict__ partial, int slices, int co, int ci, int width, T* __restrict__ gw,
                                                        TB* __restrict__ gb) {
    __shared__ float tile[32][33];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, o0 = blockIdx.x * 32, c0 = blockIdx.y * 32;
    const long long n = (long long)co * width;
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int i = 0; i < slices; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int c = c0 + w + 8 * k;
            if (c < width && o0 + lane < co) s[k] += partial[i * n + (long long)c * co + o0 + lane];
        }
#pragma unroll
    for (int k = 0; k < 4; ++k) tile[w + 8 * k][lane] = s[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int o = o0 + w + 8 * k, c = c0 + lane;
        if (o >= co || c >= width) continue;
        const float v = tile[lane][w + 8 * k];
        if (c < ci) gw[(long long)o * ci + c] = ndc::from_f32<T>(v);
        else gb[o] = ndc::from_f32<TB>(v);
    }
}

struct Plan { int ct, tiles_o, tiles_c; long long steps; Passes passes; };

// Inputs in equal tiles; slices for a CTA per multiprocessor, of at least 512 positions.
Plan plan(int batch, int co, int ci, long long n, int positions, int32_t dtype) {
    Plan p;
    p.tiles_o = (co + MT - 1) / MT;
    p.tiles_c = (ci + kMostColumns - 17) / (kMostColumns - 16);
    p.ct = ((ci + p.tiles_c - 1) / p.tiles_c + 15) / 16 * 16;
    p.steps = (long long)batch * ((n + positions - 1) / positions);
    const long long tiles = (long long)p.tiles_o * p.tiles_c;
    long long slices = std::max(1LL, std::min(ndc::num_sms() / tiles, (p.steps * positions + 511) / 512));
    const int chain = dtype == NDC_F32 ? kChain : kChain16, terms = dtype == NDC_F32 ? 3 : 1;
    const long long most = (long long)chain / (positions / 16) * leading_of(columns_of(p.ct), terms);          // steps
    if (slices * most < p.steps) {        // more slices than the GPU has room for at once: the ones that fit the same rounds of CTAs
        slices = (p.steps + most - 1) / most;
        const long long sms = ndc::num_sms(), rounds = (slices * tiles + sms - 1) / sms;
        slices = std::max(slices, rounds * sms / tiles);      // (256 -> 1000) x 2^20 in bfloat16: 27 slices 1068 us, 22 1265, 9 1080
    }
    p.passes = plan_passes(slices, (size_t)co * (ci + 1) * sizeof(float), tiles);
    return p;
}

bool too_large(int batch, int co, int ci, long long n) {
    return n > 0x7fffffffLL - 2 * KP || (long long)batch * std::max(ci, co) > 0x7fffffffLL - MT || (n + KP - 1) / KP > 0x7fffffffLL / batch ||
           ci > 65535 * (kMostColumns - 16) || (long long)co * (ci + 1LL) > (1LL << 35);
}

// Rows of n bfloat16 values, boxes of 128 rows of 64.
bool make_gradient_map(CUtensorMap& map, const void* gy, long long rows, long long n) {
    const EncodeTiled fn = encode_tiled();
    const cuuint64_t dims[2] = {(cuuint64_t)n, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)(2 * n)};
    const cuuint32_t boxes[2] = {KP, MT}, ones[2] = {1, 1};
    return fn && fn(&map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(gy), dims, strides, boxes, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool vectors(long long n, int32_t dtype, const void* gy) { return n % (dtype == NDC_BF16 ? 8 : 4) == 0 && ((uintptr_t)gy & 15) == 0; }
int positions_of(int32_t dtype, bool vec) { return dtype == NDC_BF16 && vec ? Step<bf16, true>::POSITIONS : KP; }

template <typename T, bool VEC>
cudaError_t launch(const WgradArgs& A, const Plan& p, cudaStream_t st) {
    typedef Step<T, VEC> S;
    auto kern = wgrad_kernel<T, VEC>;
    const cudaError_t e = ndc::allow_smem(kern);
    if (e != cudaSuccess) return e;
    const int stages = stages_of<S>(p.ct);
    CUtensorMap map{};
    if (S::TMA && !make_gradient_map(map, A.gy, (long long)A.steps / A.steps_n * A.co, A.n)) return cudaErrorInvalidValue;
    kern<<<dim3(p.tiles_o, p.tiles_c, p.passes.each), kThreads, 1024 + kHeader + (size_t)stages * S::bytes(columns_of(p.ct)), st>>>(map, A, stages);
    ndc::launched();
    return cudaGetLastError();
}

template <typename T, typename TB>
void launch_sum(const WgradArgs& A, const float* partial, int slices, void* gw, void* gb, cudaStream_t st) {
    const long long n = (long long)A.co * A.width;
    // a chain of up to 16 loads per thread is no longer than the other kernel's, as soon as the elements fill the GPU
    if (slices <= 16 && n >= 65536 && A.width <= 32 * 65535)
        wgrad_few_kernel<T, TB><<<dim3((A.co + 31) / 32, (A.width + 31) / 32), 256, 0, st>>>(partial, slices, A.co, A.ci, A.width, (T*)gw, (TB*)gb);
    else wgrad_sum_kernel<T, TB><<<(unsigned)((n + 31) / 32), 256, 0, st>>>(partial, slices, A.co, A.ci, A.width, (T*)gw, (TB*)gb);
    ndc::launched();
}

}  // namespace
}  // namespace q8
}  // namespace ndc

using namespace ndc::q8;

extern "C" {

size_t ndc_q8_wgrad_workspace_bytes(int32_t batch, int32_t co, int32_t ci, int64_t n, int32_t dtype) {
    if (batch <= 0 || co <= 0 || ci <= 0 || n <= 0 || too_large(batch, co, ci, n)) return 0;
    // the most that either step asks for
    return std::max(plan(batch, co, ci, n, KP, dtype).passes.places(), plan(batch, co, ci, n, 2 * KP, dtype).passes.places()) * co * (ci + 1) * sizeof(float);
}

int ndc_q8_wgrad(int32_t batch, int32_t co, int32_t ci, int64_t n, int32_t dtype, const void* gy, const void* values, const void* scales,
                 void* gw, void* gb, int32_t gb_dtype, void* workspace, size_t workspace_bytes, void* stream) {
    if (!gy || !values || !scales || !gw) return fail(NDC_ERR_INVALID, "q8 weight gradient: gy, values, scales and gw must not be NULL");
    if (batch <= 0 || co <= 0 || ci <= 0 || n <= 0) return fail(NDC_ERR_INVALID, "q8 weight gradient: extents must be positive");
    if ((dtype != NDC_F32 && dtype != NDC_BF16) || (gb && gb_dtype != NDC_F32 && gb_dtype != NDC_BF16))
        return fail(NDC_ERR_INVALID, "q8 weight gradient: dtype must be NDC_F32 or NDC_BF16");
    if ((uintptr_t)values & 15) return fail(NDC_ERR_ALIGNMENT, "q8 weight gradient: values must lie on 16 bytes");
    if (off_elements(dtype, {gy, gw}) || off_elements(gb_dtype, {gb}) || off_elements(NDC_F32, {workspace}))
        return fail(NDC_ERR_ALIGNMENT, "q8 weight gradient: a tensor does not lie on its elements' size");
    const bool vec = vectors(n, dtype, gy);
    const int positions = positions_of(dtype, vec);
    if (too_large(batch, co, ci, n)) return fail(NDC_ERR_UNSUPPORTED, "q8 weight gradient: problem too large");
    const Plan p = plan(batch, co, ci, n, positions, dtype);
    const size_t need = ndc_q8_wgrad_workspace_bytes(batch, co, ci, n, dtype);
    if (!workspace || workspace_bytes < need) return fail(NDC_ERR_WORKSPACE, "q8 weight gradient: workspace of %zu bytes needed", need);
    if (ndc::tc::take_expired()) return fail(NDC_ERR_TIMEOUT, "a wait inside a kernel of an earlier call ran out after one second");
    const int width = ci + (gb ? 1 : 0);
    const size_t place = (size_t)co * width;
    float* const places = (float*)workspace;
    WgradArgs A{gy, (const unsigned char*)values, (const unsigned char*)scales, places + p.passes.first() * place, n, pitch_of(n), (int)scales_of(n), co, ci, p.ct,
                width, (int)((n + positions - 1) / positions), p.steps, p.passes.slices, 0, nullptr};
    cudaError_t e = ndc::tc::expired_word(A.expired);
    if (e != cudaSuccess) return fail(NDC_ERR_CUDA, "q8 weight gradient: %s", cudaGetErrorString(e));
    cudaStream_t st = (cudaStream_t)stream;
    for (int i = 0; i < p.passes.count() && e == cudaSuccess; ++i) {
        A.slice0 = i * p.passes.each;
        if (dtype == NDC_F32) e = vec ? launch<float, true>(A, p, st) : launch<float, false>(A, p, st);
        else e = vec ? launch<bf16, true>(A, p, st) : launch<bf16, false>(A, p, st);
        if (e != cudaSuccess) break;
        const float* from = places + p.passes.from(i) * place;
        const int added = p.passes.added(i);
        if (i + 1 < p.passes.count()) {
            if (ndc_proj_sum(added, (int64_t)place, NDC_F32, from, places + p.passes.to(i) * place, stream) != NDC_OK)
                return fail(NDC_ERR_CUDA, "q8 weight gradient: %s", ndc_proj_last_error());
            continue;
        }
        const bool wide = gb && gb_dtype == NDC_F32;
        if (dtype == NDC_F32) { if (gb && !wide) launch_sum<float, bf16>(A, from, added, gw, gb, st); else launch_sum<float, float>(A, from, added, gw, gb, st); }
        else if (wide) launch_sum<bf16, float>(A, from, added, gw, gb, st);
        else launch_sum<bf16, bf16>(A, from, added, gw, gb, st);
        e = cudaGetLastError();
    }
    return e == cudaSuccess ? NDC_OK : fail(NDC_ERR_CUDA, "q8 weight gradient: %s", cudaGetErrorString(e));
}

}  // extern "C"
