// Lines "len n window" on standard input -> "start tiles sees..." for the entries around each row's borders.  Built with signed overflow as an error.
#include <cstdio>

#include "paged_span.h"

int main() {
    int len, n, window;
    while (std::scanf("%d %d %d", &len, &n, &window) == 3) {
        const cd::PaSpan s = cd::pa_span(len, n, window);
        std::printf("%d %d", s.start, s.tiles);
        for (int j = 0; j < n; j += n > 8 ? n / 8 : 1) {
            const int last = len - n + j;
            const long long near[] = {0, (long long)last - window, (long long)last - window + 1, (long long)last - 1, last, (long long)last + 1, (long long)len - 1};
            for (long long t : near) std::printf(" %d", t >= 0 && t < len ? (int)cd::pa_sees((int)t, last, window) : 2);
        }
        std::printf("\n");
    }
}
