// Which of a sequence's cache entries its new rows see (paged_attn.cuh).  On the host too, so that its arithmetic is tested there: no
// step of it leaves 32 bits, whatever the length (below 2^31 - 1024), the rows and the window (up to 2^31 - 1).
#pragma once

#if defined(__CUDACC__)
#define PA_BOTH __host__ __device__
#else
#define PA_BOTH
#endif

namespace cd {

constexpr int PA_TILE = 64;  // entries

struct PaSpan {
    int start, tiles;  // the first tile's first entry; tiles up to the sequence's end, none where there are no rows or no entries
};
// Row j of n sees entries up to len - n + j, with a window the last `window` of them: the first row's are the first ones any row sees.
PA_BOTH inline PaSpan pa_span(int len, int n, int window) {
    PaSpan s{0, 0};
    const int up_to = len - n + 1;  // entries up to the first row's own; not positive where there are more rows than entries
    if (window > 0 && up_to > window) s.start = (up_to - window) & ~(PA_TILE - 1);
    if (n > 0 && len > 0) s.tiles = (len - s.start + PA_TILE - 1) / PA_TILE;
    return s;
}
// whether a row whose own entry is `last` (negative: it has none) sees entry t
PA_BOTH inline bool pa_sees(int t, int last, int window) { return t <= last && (window == 0 || last - t < window); }

}  // namespace cd
