// The ranges of keys that the eviction's search goes through; host and device, so that it can be tested without a GPU.
#pragma once

#include <bit>
#include <cstdint>

namespace w4 {

constexpr int kEvictBins = 2048;
constexpr uint32_t kEvictFirst = 0xAF800000u;     // key of 2^-32
constexpr int kEvictFirstShift = 18;

// Keys first .. last, in bins of 2^shift.  In the first round (clamp) the bins at the ends hold all keys beyond them too.
struct KeyRange {
    uint32_t first = kEvictFirst, last = kEvictFirst + (static_cast<uint32_t>(kEvictBins) << kEvictFirstShift) - 1;
    int shift = kEvictFirstShift;
    bool clamp = true;
};
// The range of one bin of a range.  The last bin may reach beyond the range, where there are keys that an earlier round has
// counted: it ends with the range.
constexpr KeyRange narrowed(const KeyRange& r, uint32_t bin) {
    const uint32_t at = r.first + (bin << r.shift), span = (1u << r.shift) - 1u;
    KeyRange n;
    n.first = r.clamp && bin == 0 ? 0u : at;
    n.last = r.clamp && bin == kEvictBins - 1 ? ~0u : r.last - at < span ? r.last : at + span;
    const uint32_t wide = (n.last - n.first) / kEvictBins;
#ifdef __CUDA_ARCH__
    n.shift = 32 - __clz(wide);
#else
    n.shift = std::bit_width(wide);
#endif
    n.clamp = false;
    return n;
}

}  // namespace w4
