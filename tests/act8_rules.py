"""The rules by which calls on 8-bit activations are cut (ek_internal.h), compiled for the host: tests ask them which kernel a
call takes instead of restating them."""
import os
import shutil
import subprocess
import tempfile

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INCLUDE = "/opt/rocm/include"

SOURCE = r'''
#include "ek_internal.h"
#include <cstdio>
int main()
{
    char what[16];
    while (scanf("%15s", what) == 1) {
        long long a, b, c, d, n;
        if (what[0] == 'b') {                    // batch of calls: hidden inter n_calls rows...
            if (scanf("%lld %lld %lld", &a, &b, &n) != 3) return 1;
            ek::Q8Batch q;
            for (long long i = 0; i < n; ++i) { if (scanf("%lld", &c) != 1) return 1; q.add(c); }
            printf("%d\n", (int)q.streamed(a, b));
        } else if (what[0] == 'e') {             // one expert's call: rows hidden inter
            if (scanf("%lld %lld %lld", &n, &a, &b) != 3) return 1;
            printf("%d\n", (int)(n <= 16 || ek::q8_wide_cut_pays(n, ek::q8_items((int)n), n, a, b)));
        } else if (what[0] == 'i') {             // items of a segment of n rows
            if (scanf("%lld", &n) != 1) return 1;
            const int items = ek::q8_items((int)n);
            for (int i = 0; i < items; ++i) {
                int first, rows;
                ek::q8_item((int)n, items, i, &first, &rows);
                printf("%d %d ", first, rows);
            }
            printf("\n");
        } else if (what[0] == 'c') {             // a layer call: pairs experts hidden inter
            if (scanf("%lld %lld %lld %lld", &a, &b, &c, &d) != 4) return 1;
            const int k = ek::q8_one_class(a, b, c, d);
            printf("%d %lld %lld\n", k, (long long)ek::list_capacity(ek::kListStream, a, b, k), (long long)ek::list_capacity(ek::kListT128, a, b, k));
        } else {                                 // a dense product: rows K N
            if (scanf("%lld %lld %lld", &n, &a, &b) != 3) return 1;
            printf("%d\n", (int)(n <= 16 || ek::q8_stream_us(n, a, b) < ek::q8_tile_us(n, a, b)));
        }
    }
}
'''
_exe = None


def available():
    return bool(shutil.which("g++")) and os.path.exists(os.path.join(INCLUDE, "hip", "hip_runtime.h"))


def ask(lines):
    """One list of numbers per question."""
    global _exe
    if _exe is None:
        d = tempfile.mkdtemp(prefix="act8_rules")
        src, exe = os.path.join(d, "rules.cpp"), os.path.join(d, "rules")
        with open(src, "w") as f:
            f.write(SOURCE)
        subprocess.run(["g++", "-D__HIP_PLATFORM_AMD__", "-std=c++17", "-O1", "-I", INCLUDE, "-I", os.path.join(ROOT, "expert-kit_amd", "csrc"), src,
                        "-o", exe], check=True, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, timeout=300)
        _exe = exe
    out = subprocess.run([_exe], input="\n".join(lines) + "\n", stdout=subprocess.PIPE, text=True, check=True, timeout=60).stdout
    return [[int(v) for v in line.split()] for line in out.strip("\n").split("\n")]


def dense_streams(n, K, N):
    """Whether a dense product takes the streaming kernel (else the tile kernel)."""
    return bool(ask([f"d {n} {max((K + 63) // 64 * 64, 128)} {(N + 15) // 16 * 16}"])[0][0])


def layer_class(pairs, experts, hidden, inter):
    return ask([f"c {pairs} {experts} {hidden} {inter}"])[0][0]


def expert_streams(n, hidden, inter):
    return bool(ask([f"e {n} {hidden} {inter}"])[0][0])


def batch_streams(rows, hidden, inter):
    return bool(ask([f"b {hidden} {inter} {len(rows)} " + " ".join(map(str, rows))])[0][0])
