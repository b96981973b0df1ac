// Lists of tensors on the host, ahead of launches that take several of them: no device code, nothing of HIP.
#pragma once
#include <stdint.h>

#include <algorithm>

#include "../../include/coat_hip.h"

// Blocks of `threads` that a launch takes in one dimension: HIP has fewer than 2^32 threads there.
constexpr int64_t coat_max_blocks(int threads) { return 0xffffffffll / threads; }

// Calls fn(first, last, chunks) for each run of tensors that one launch takes: at most `most` tensors that are not empty and
// `most_chunks` chunks of `chunk` elements.  Returns COAT_ESHAPE if one tensor alone has more.
template <typename F>
static int coat_for_each_launch(int count, const int64_t* numel, int64_t chunk, int most, int64_t most_chunks, F fn) {
    for (int i = 0; i < count;) {
        const int first = i;
        int used = 0;
        int64_t chunks = 0;
        for (; i < count && used < most; i++) {
            if (numel[i] == 0) continue;
            const int64_t c = (numel[i] + chunk - 1) / chunk;
            if (chunks + c > most_chunks) {
                if (used == 0) return COAT_ESHAPE;
                break;
            }
            chunks += c;
            used++;
        }
        if (used == 0) break;  // only empty tensors were left
        if (const int rc = fn(first, i, chunks)) return rc;
    }
    return COAT_OK;
}

// Whether a tensor that is written shares memory with another tensor.  The spans are sorted here.
struct CoatSpan {
    uintptr_t begin, end;
    bool written;
};
static inline bool coat_overlap(CoatSpan* spans, size_t n) {
    std::sort(spans, spans + n, [](const CoatSpan& a, const CoatSpan& b) { return a.begin < b.begin; });
    uintptr_t end_any = 0, end_written = 0;
    for (size_t i = 0; i < n; i++) {
        if (spans[i].begin < (spans[i].written ? end_any : end_written)) return true;
        if (spans[i].end > end_any) end_any = spans[i].end;
        if (spans[i].written && spans[i].end > end_written) end_written = spans[i].end;
    }
    return false;
}
