// What the units of the 8-bit calls share on the host: their error text and a check of pointers.
#pragma once

#include <algorithm>
#include <cstdint>
#include <initializer_list>

#include "ndc_b200.h"
#include "ndc_common.cuh"

namespace ndc {
namespace q8 {

// Sets the message of ndc_q8_last_error and returns `status`.
int fail(int status, const char* fmt, ...);

// Whether one of the tensors does not lie on a multiple of its elements' size.
inline bool off_elements(int32_t dtype, std::initializer_list<const void*> tensors) {
    for (const void* p : tensors)
        if ((uintptr_t)p & (dtype == NDC_F32 ? 3 : 1)) return true;
    return false;
}

// A sum in slices, whose float32 partial sums lie in places one after the other.  Where they would be more memory than that, it takes
// launches of `each` slices: a launch's partial sums and what the ones before it came to are added up into a place before or behind
// them in turn.
struct Passes {
    int slices, each;
    int count() const { return slices / each; }
    size_t places() const { return count() > 1 ? (size_t)each + 2 : slices; }
    size_t first() const { return count() > 1; }                            // place of a launch's slices
    // of launch i: the places that are added up, and where to (the last launch's go to the result)
    size_t from(int i) const { return i % 2 ? 0 : first(); }
    int added(int i) const { return each + (i > 0); }
    size_t to(int i) const { return i % 2 ? (size_t)each + 1 : 0; }
};

// `bytes` of a place, `tiles` of results (CTAs of a slice).  64 MiB: slices that share a launch's time alone, one or two CTAs to a multiprocessor
// and up to three rounds of them, stay below that; sums of long chains do not.  2 x (512 -> 2048) channels x 64^3 positions in float32 took 2.1 GB of
// partial sums, where the checkpoint saves 0.8: now 59 MB, and 6.8 ms for 6.1 (with 128 MiB 7.4, the partial sums no longer in the L2 cache).
// Launches have whole rounds of CTAs, as nearly as slices make them.
inline Passes plan_passes(long long slices, size_t bytes, long long tiles) {
    constexpr long long kMostBytes = 64LL << 20, kMostSlices = 65535;
    const long long places = std::min(kMostSlices, kMostBytes / (long long)bytes);
    if (slices <= std::max(1LL, places)) return {(int)slices, (int)slices};
    long long each = std::max(1LL, places - 2);
    const long long sms = num_sms(), most = each;
    auto filled = [&](long long e) { return (double)(e * tiles) / (double)((e * tiles + sms - 1) / sms * sms); };
    if (most * tiles < 16 * sms)
        for (long long e = most; 2 * e > most; --e)
            if (filled(e) > filled(each) + 0.01) each = e;
    return {(int)((slices + each - 1) / each * each), (int)each};
}

}  // namespace q8
}  // namespace ndc
