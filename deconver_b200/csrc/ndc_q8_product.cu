// Products of operands held in 8 bits (format: ndc_q8.cuh) on the 5th-generation tensor cores:
//
//     D[i, j] = sum over k of A[i, k] B[j, k],      A, B: e4m3 rows along k, a power of two per 128 of them
//
// The powers of two are the block scales of `tcgen05.mma kind::mxf8f6f4` (UE8M0, one for 32 elements of a row
// and so four times the same one here): the tensor core applies them to the products, and no
// partial sum leaves its accumulators to be scaled.  All sums are float32 in TMEM.
//
// A CTA has a tile of 128 x NT results.  Stages of 128 elements along k come by TMA into shared memory in the
// 128-byte swizzle; two warps bring the scales, a byte per row, as whole words of four blocks (the MMA
// picks one of the four), transposed to the 32 x 16 bytes that tcgen05.cp spreads over the lanes of TMEM.  Rows
// past the end of a tensor are zero or another sample's: they give rows and columns of D that are not stored.
//
// D goes out transposed: D[i, j] to out[(i / rows) * cols * rows + j * rows + i % rows].  With positions as
// rows that is the channels-first layout; a thread has a row, so a warp's 32 stores of a column
// are neighbours (10 of the 86 us below).
//
// 65536 x 512 of 2048 in bfloat16: 86 us, 1600 TFLOP/s of 3310.  A step of 128 x 256 results takes 0.75 us, its MMAs half of that: what
// bounds it are its 48 KB from the L2 cache (9.5 TB/s over all), and at 8 steps the 3.4 us before and after them.
#include <algorithm>

#include "ndc_b200.h"
#include "ndc_common.cuh"
#include "ndc_q8.cuh"
#include "ndc_q8_host.h"
#include "ndc_q8_mma.cuh"
#include "ndc_tc_host.h"

namespace ndc {
namespace q8 {
namespace {

using namespace ndc::tc;
typedef __nv_bfloat16 bf16;

constexpr int kThreads = 256;          // four warps for the results, then one each for TMA, MMA and the scales of A and B

struct ProductArgs {
    const unsigned char *sa, *sb;      // scales
    int pitch_a, pitch_b;              // of a row's scales
    long long rows_a, rows_b;          // of the tensors
    int m, n, k;                       // of the product; k: of one sample
    int samples, kblocks;              // k runs over samples of kblocks blocks; sample s begins at row s * m of A, s * n of B
    int slices, slice0;                // of that sequence of blocks; the launch's first one
    const void* bias;                  // per column, float32 or bfloat16, or NULL
    int bias_bf16;
    void* out;                         // per slice m * n
    long long rows;                    // of D that lie next to each other
    unsigned* expired;
};

template <int NT> struct Shape {
    static constexpr int SFB = (NT + 127) / 128;                  // 128-row groups of B's scales
    static constexpr int STAGES = NT == 256 ? 4 : 3;
    static constexpr int BYTES = MT * KT + NT * KT;               // of a stage's operands
    static constexpr int SF_BYTES = 512 * (1 + SFB);
    static constexpr int HEADER = 2048;                           // barriers, the TMEM address, the bias
    static constexpr int COLS = NT + STAGES * 4 * (1 + SFB);
    static constexpr int TMEM = COLS <= 64 ? 64 : COLS <= 128 ? 128 : COLS <= 256 ? 256 : 512;
    static constexpr size_t SMEM = 1024 + HEADER + STAGES * (BYTES + SF_BYTES);
};

template <int NT, typename T>
__global__ void __launch_bounds__(kThreads) product_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                                                           const __grid_constant__ ProductArgs P) {
    using S = Shape<NT>;
    extern __shared__ unsigned char raw_smem[];
    unsigned char* smem = raw_smem + ((1024u - (smem_u32(raw_smem) & 1023u)) & 1023u);
    const unsigned base = smem_u32(smem);
    const unsigned full = base, empty = base + 8 * S::STAGES, done = base + 16 * S::STAGES, slot = done + 8;
    float* bias = reinterpret_cast<float*>(smem + 256);
    const unsigned stages = base + S::HEADER, scales = stages + S::STAGES * S::BYTES;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // tiles of the same rows of A run at the same time (one after the other, 65536 x 512 of 2048 took 94 us for 86)
    const unsigned tiles_n = (P.n + NT - 1) / NT;
    const int n0 = blockIdx.x % tiles_n * NT, cols = min(NT, P.n - n0);
    const long long m0 = (long long)(blockIdx.x / tiles_n) * MT;
    const long long total = (long long)P.samples * P.kblocks;
    const long long slice = P.slice0 + (int)blockIdx.z;
    const int first = (int)(total * slice / P.slices), steps = (int)(total * (slice + 1) / P.slices) - first;

    if (threadIdx.x == 0) {
        for (int s = 0; s < S::STAGES; ++s) { mbar_init(full + 8 * s, 3); mbar_init(empty + 8 * s, 1); }
        mbar_init(done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) tmem_alloc(slot, S::TMEM);
    for (int j = threadIdx.x; j < NT; j += kThreads) bias[j] = P.bias && j < cols ? load_bias(P.bias, P.bias_bf16, n0 + j) : 0.0f;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const unsigned tmem = *reinterpret_cast<volatile unsigned*>(smem + (slot - base));
    bool ok = true;

    if (warp == 4) {
        if (lane == 0) {
            int issued = 0;
            for (int t = 0; t < steps && ok; ++t) {
                const int s = t % S::STAGES;
                if (t >= S::STAGES) ok = mbar_wait_thread(empty + 8 * s, (t / S::STAGES - 1) & 1, kWaitLimit);
                if (!ok) break;
                const int it = first + t, sample = it / P.kblocks, kb = it - sample * P.kblocks;
                const unsigned at = stages + s * S::BYTES;
                expect_bytes(full + 8 * s, S::BYTES);
                tma_load(at, &map_a, kb * KT, (int)(m0 + (long long)sample * P.m), full + 8 * s);
                tma_load(at + MT * KT, &map_b, kb * KT, n0 + sample * P.n, full + 8 * s);
                ++issued;
            }
            if (!ok)       // the copies that are on their way
                for (int t = max(0, issued - S::STAGES); t < issued; ++t) mbar_wait_thread(full + 8 * (t % S::STAGES), (t / S::STAGES) & 1, kWaitLimit);
        }
    } else if (warp == 5) {
        if (elect()) {
            int kb = first % P.kblocks;
            for (int t = 0; t < steps; ++t) {
                const int s = t % S::STAGES;
                ok = mbar_wait_thread(full + 8 * s, (t / S::STAGES) & 1, kWaitLimit);
                if (!ok) break;
                tc_fence_after();
                const unsigned sfa = tmem + NT + s * 4 * (1 + S::SFB), sfb = sfa + 4, from = scales + s * S::SF_BYTES;
                const unsigned long long a = swizzled_desc(stages + s * S::BYTES), b = swizzled_desc(stages + s * S::BYTES + MT * KT);
                const unsigned idesc = scaled_instr((cols + 15) / 16 * 16, kb & 3, kb & 3);
                const int parts = (P.k - kb * KT + 31) / 32;
                {
                    scales_to_tmem(sfa, mat_desc(from, 128, 128));
#pragma unroll
                    for (int g = 0; g < S::SFB; ++g) scales_to_tmem(sfb + 4 * g, mat_desc(from + 512 * (1 + g), 128, 128));
#pragma unroll
                    for (int i = 0; i < KT / 32; ++i)
                        if (i < parts) mma_scaled(tmem, a + 2 * i, b + 2 * i, idesc, sfa, sfb, t > 0 || i > 0);
                    mma_commit(empty + 8 * s);
                }
                if (++kb == P.kblocks) kb = 0;
            }
            mma_commit(done);
        }
    } else if (warp >= 6) {
        // 128 rows of A, or NT of B: lane l has rows l, l + 32, l + 64 and l + 96 of a group
        const bool is_a = warp == 6;
        const unsigned char* table = is_a ? P.sa : P.sb;
        const int pitch = is_a ? P.pitch_a : P.pitch_b, groups = is_a ? 1 : S::SFB;
        const long long last = (is_a ? P.rows_a : P.rows_b) - 1;
        for (int t = 0; t < steps && ok; ++t) {
            const int s = t % S::STAGES, it = first + t, sample = it / P.kblocks, kb = it - sample * P.kblocks;
            const long long row = is_a ? m0 + (long long)sample * P.m : n0 + (long long)sample * P.n;
            unsigned w[S::SFB][4];
#pragma unroll
            for (int g = 0; g < S::SFB; ++g)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (g < groups)
                        w[g][i] = __ldg(reinterpret_cast<const unsigned*>(table + min(last, row + 128 * g + 32 * i + lane) * pitch + (kb & ~3)));
            if (t >= S::STAGES) ok = mbar_wait(empty + 8 * s, (t / S::STAGES - 1) & 1);
            if (!ok) break;
#pragma unroll
            for (int g = 0; g < S::SFB; ++g)
                if (g < groups)
                    *reinterpret_cast<uint4*>(smem + (scales - base) + s * S::SF_BYTES + 512 * (is_a ? 0 : 1 + g) + 16 * lane) =
                        make_uint4(w[g][0], w[g][1], w[g][2], w[g][3]);
            fence_async_proxy();
            __syncwarp();
            if (lane == 0) mbar_arrive(full + 8 * s);
        }
    }
    // The results, by all warps: two have each 32 rows.  (Four of them alone took 6 us more at 65536 x 512 of 2048)
    {
        ok = __all_sync(0xffffffffu, ok);
        if (ok) ok = mbar_wait(done, 0);
        tc_fence_after();
        const int quarter = warp & 3;
        const long long i = m0 + 32 * quarter + lane;
        const long long group = i / P.rows, rest = i - group * P.rows;
        T* out = reinterpret_cast<T*>(P.out) + (long long)blockIdx.z * P.m * P.n + (group * P.n + n0) * P.rows + rest;
        const bool in = i < P.m && ok;
#pragma unroll 1
        for (int j0 = 32 * (warp >> 2); j0 < cols; j0 += 64) {
            float v[32];
            __syncwarp();
            tmem_load32(tmem + ((unsigned)(32 * quarter) << 16) + j0, v);
            store_columns(out + j0 * P.rows, P.rows, v, cols - j0, in, bias[j0 + lane], P.bias != nullptr);
        }
        tc_fence_before();
    }
    if (!ok) report_expired(P.expired);
    __syncthreads();
    if (warp == 0) {
        tc_fence_after();
        tmem_free(tmem, S::TMEM);
    }
}

// ---- host -------------------------------------------------------------------------------------

template <int NT, typename T>
cudaError_t launch(const CUtensorMap& a, const CUtensorMap& b, const ProductArgs& P, int slices, cudaStream_t st) {
    auto kern = product_kernel<NT, T>;
    const cudaError_t e = ndc::allow_smem(kern);
    if (e != cudaSuccess) return e;
    kern<<<dim3((unsigned)((P.m + MT - 1) / MT) * (unsigned)((P.n + NT - 1) / NT), 1, (unsigned)slices), kThreads, Shape<NT>::SMEM, st>>>(a, b, P);
    ndc::launched();
    return cudaGetLastError();
}

// Columns of a tile: 256 halve what comes from the L2 cache for each row, if they leave a CTA for each multiprocessor.
int columns_of(long long m, long long n, long long slices) {
    if (n <= 64) return 64;
    const long long tiles = ((m + MT - 1) / MT) * ((n + 255) / 256) * slices;
    return n <= 128 || tiles < ndc::num_sms() ? 128 : 256;
}

// Slices of the sum along k, of four blocks at least: the ones of the least time by rounds of CTAs, one or two to a multiprocessor.  A
// step of 256 columns counts 1 (0.45 us), one of 128 or 64, at two CTAs each, 1.1 and 0.8; what comes before and after the steps
// counts 9 and 6, a launch to add slices up 6, and a slice's results are written and read.  At 2048 x 512 of 65536 (all slices
// and their sum) 4 slices take 75 us, 5 106, 7 88 and 9 73; the model says 73, 108, 84 and 71.  2048 x 512 of 1024 takes 7 us in
// one slice, 11 in two.  For float32 results a slice has 32 blocks at most: the MMA cuts its sums off, and a chain of 128 shrinks
// by 128 2^-25 to 128 2^-24; for bfloat16 ones 256, 2^-14.
Passes plan_slices(int samples, long long m, long long n, long long k, int32_t dtype) {
    const long long total = (long long)samples * ((k + KT - 1) / KT), chain = dtype == NDC_F32 ? 32 : 256, least = (total + chain - 1) / chain, most = std::max(least, (total + 3) / 4);
    long long best = least;
    double best_time = 1e300;
    auto consider = [&](long long slices) {
        slices = std::max(least, std::min(slices, most));
        const int nt = columns_of(m, n, slices), resident = nt == 256 ? 1 : 2;
        const long long ctas = ((m + MT - 1) / MT) * ((n + nt - 1) / nt) * slices, rounds = (ctas + resident * ndc::num_sms() - 1) / (resident * ndc::num_sms());
        const double step = nt == 256 ? 1.0 : nt == 128 ? 1.1 : 0.8, rest = nt == 256 ? 9.0 : 6.0;
        const double time = (double)rounds * ((double)((total + slices - 1) / slices) * step + rest) + (slices > 1 ? 6.0 + 2e-6 * (double)slices * (double)m * (double)n : 0.0);
        if (time < best_time) { best_time = time; best = slices; }
    };
    consider(least);
    for (int width = 128; width <= 256; width *= 2)           // the largest ones that fit so many rounds
        for (int rounds = 1; rounds <= 3; ++rounds) {
            const int nt = n <= 64 ? 64 : width;
            consider((long long)rounds * (nt == 256 ? 1 : 2) * ndc::num_sms() / (((m + MT - 1) / MT) * ((n + nt - 1) / nt)));
        }
    const int nt = columns_of(m, n, best);
    return plan_passes(best, (size_t)(m * n) * sizeof(float), ((m + MT - 1) / MT) * ((n + nt - 1) / nt));
}

bool too_large(int samples, long long m, long long n, long long k) {
    return m > (0x7fffffffLL - 4 * MT) / samples || n > (0x7fffffffLL - 4 * MT) / samples || k > 0x7fffffffLL - KT || (k + KT - 1) / KT > 0x7fffffffLL / samples ||
           (m + MT - 1) / MT > 0x7fffffffLL / ((n + 63) / 64);
}

}  // namespace
}  // namespace q8
}  // namespace ndc

using namespace ndc::q8;

extern "C" {

size_t ndc_q8_product_workspace_bytes(int32_t samples, int64_t m, int64_t n, int64_t k, int32_t dtype) {
    if (samples <= 0 || m <= 0 || n <= 0 || k <= 0 || too_large(samples, m, n, k)) return 0;
    return plan_slices(samples, m, n, k, dtype).places() * m * n * sizeof(float);
}

int ndc_q8_product(int32_t samples, int64_t m, int64_t n, int64_t k, int32_t dtype, const void* a_values, const void* a_scales,
                   const void* b_values, const void* b_scales, const void* bias, int32_t bias_dtype, int64_t rows, void* out, void* workspace,
                   size_t workspace_bytes, void* stream) {
    if (!a_values || !a_scales || !b_values || !b_scales || !out) return fail(NDC_ERR_INVALID, "q8 product: operands and out must not be NULL");
    if (samples <= 0 || m <= 0 || n <= 0 || k <= 0 || rows <= 0 || m % rows) return fail(NDC_ERR_INVALID, "q8 product: extents must be positive, m a multiple of rows");
    if ((dtype != NDC_F32 && dtype != NDC_BF16) || (bias && bias_dtype != NDC_F32 && bias_dtype != NDC_BF16)) return fail(NDC_ERR_INVALID, "q8 product: dtype must be NDC_F32 or NDC_BF16");
    if (too_large(samples, m, n, k)) return fail(NDC_ERR_UNSUPPORTED, "q8 product: problem too large");
    for (const void* p : {a_values, b_values})
        if ((uintptr_t)p & 15) return fail(NDC_ERR_ALIGNMENT, "q8 product: values must lie on 16 bytes");
    for (const void* p : {a_scales, b_scales})
        if ((uintptr_t)p & 3) return fail(NDC_ERR_ALIGNMENT, "q8 product: scales must lie on 4 bytes");
    if (off_elements(dtype, {out}) || off_elements(bias_dtype, {bias}) || off_elements(NDC_F32, {workspace}))
        return fail(NDC_ERR_ALIGNMENT, "q8 product: out, bias or workspace misaligned");
    const bool split = samples > 1 || workspace;       // a sum over samples, or a long one, in slices
    if (split && (bias || rows != m)) return fail(NDC_ERR_INVALID, "q8 product: slices have neither bias nor groups of rows");
    const Passes passes = split ? plan_slices(samples, m, n, k, dtype) : Passes{1, 1};
    const int slices = passes.slices;
    const size_t need = passes.places() * m * n * sizeof(float);
    if (split && (!workspace || workspace_bytes < need)) return fail(NDC_ERR_WORKSPACE, "q8 product: workspace of %zu bytes needed", need);
    if (ndc::tc::take_expired()) return fail(NDC_ERR_TIMEOUT, "a wait inside a kernel of an earlier call ran out after one second");
    ProductArgs P{};
    P.sa = (const unsigned char*)a_scales; P.sb = (const unsigned char*)b_scales;
    P.pitch_a = P.pitch_b = (int)scales_of(k);
    P.rows_a = (long long)samples * m; P.rows_b = (long long)samples * n;
    P.m = (int)m; P.n = (int)n; P.k = (int)k;
    P.samples = samples; P.kblocks = (int)((k + KT - 1) / KT); P.slices = slices;
    P.bias = bias; P.bias_bf16 = bias_dtype == NDC_BF16; P.out = slices > 1 ? (float*)workspace + passes.first() * m * n : out; P.rows = rows;
    cudaError_t e = ndc::tc::expired_word(P.expired);
    if (e != cudaSuccess) return fail(NDC_ERR_CUDA, "q8 product: %s", cudaGetErrorString(e));
    const int nt = columns_of(m, n, passes.each);
    CUtensorMap a, b;
    if (!make_map(a, a_values, P.rows_a, pitch_of(k), MT) || !make_map(b, b_values, P.rows_b, pitch_of(k), nt))
        return fail(NDC_ERR_CUDA, "q8 product: the driver refused a tensor map");
    cudaStream_t st = (cudaStream_t)stream;
    auto go = [&](auto type) {
        typedef decltype(type) T;
        return nt == 64 ? launch<64, T>(a, b, P, passes.each, st) : nt == 128 ? launch<128, T>(a, b, P, passes.each, st) : launch<256, T>(a, b, P, passes.each, st);
    };
    for (int i = 0; i < passes.count(); ++i) {
        P.slice0 = i * passes.each;
        e = dtype == NDC_F32 || slices > 1 ? go(float()) : go(bf16());
        if (e != cudaSuccess) return fail(NDC_ERR_CUDA, "q8 product: %s", cudaGetErrorString(e));
        if (slices == 1) break;
        const bool last = i + 1 == passes.count();
        float* const places = (float*)workspace;
        if (ndc_proj_sum(passes.added(i), m * n, last ? dtype : NDC_F32, places + passes.from(i) * m * n, last ? out : places + passes.to(i) * m * n, stream) != NDC_OK)
            return fail(NDC_ERR_CUDA, "q8 product: %s", ndc_proj_last_error());
    }
    return NDC_OK;
}

}  // extern "C"
