"""Which entries a sequence's rows see (paged_span.h), on the CPU: at the ends of what lengths, rows and windows may be."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
MOST = 2 ** 31 - 1


def test_spans_at_the_ends_of_32_bits(tmp_path):
    exe = str(tmp_path / "check")
    subprocess.check_call(["g++", "-O1", "-std=c++17", "-fsanitize=signed-integer-overflow", "-fno-sanitize-recover=all", "-I", os.path.join(ROOT, "rustane_b200", "csrc"),
                           os.path.join(ROOT, "tests", "kernels", "paged_span_check.cpp"), "-o", exe])
    cases = [(n, rows, w) for n in (0, 1, 2, 63, 64, 65, 1000, 131072, 2 ** 31 - 1025, 2 ** 31 - 1024) for rows in (0, 1, 4, 64, 65536)
             for w in (0, 1, 2, 63, 64, 65, 1000, 2 ** 30, MOST - 65536, MOST - 1, MOST)]
    got = subprocess.run([exe], input="\n".join("%d %d %d" % c for c in cases), capture_output=True, text=True, check=True).stdout.split("\n")
    for (n, rows, w), line in zip(cases, got):
        line = [int(x) for x in line.split()]
        first = n - rows + 1 - w if w else 0  # of the first row, in integers without an end
        start = first // 64 * 64 if first > 0 else 0
        want = [start, -(-(n - start) // 64) if rows and n else 0]
        for j in range(0, rows, rows // 8 if rows > 8 else 1):
            last = n - rows + j
            for t in (0, last - w, last - w + 1, last - 1, last, last + 1, n - 1):
                want.append(2 if not 0 <= t < n else int(t <= last and (w == 0 or t > last - w)))
        assert line == want, (n, rows, w)
