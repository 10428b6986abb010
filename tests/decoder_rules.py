"""The rules by which a call of the gated feed-forward block takes its kernels (svox_amd/csrc/decoder/rules.h), compiled as they stand."""
import os
import subprocess

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "svox_amd", "csrc", "decoder", "rules.h")
PROGRAM = r"""
#include <cstdio>
#include "%s"
using namespace svox_decoder;
static const char* kNames[] = {"small", "deep", "medium", "large"};
template <int planes>
void say(const SvoxGatedFfn& s) {
    using R = Rules<planes>;
    const long long wide = up_to(s.hidden, 8);
    for (int backward = 0; backward < 2; ++backward) {
        const char* const pass = backward ? "gradients" : "forward";
        if (R::few_rows(s, backward)) printf("%%s few %%d\n", pass, s.rows <= 16 ? 1 : s.rows <= 32 ? 2 : 4);
        else if (R::narrow(s, backward)) printf("%%s narrow %%d %%d by %%d\n", pass, narrow_steps(s.dim), narrow_steps(s.out), R::narrow_tiles(s.rows));
        else {
            printf("%%s hidden %%s\n%%s result %%s\n", pass, kNames[R::hidden_size(s.rows, wide)], pass, kNames[R::output_size(s.rows, backward ? s.dim : s.out)]);
            if (backward) printf("weights %%s %%s\n", kNames[R::weight_split(s).size], R::weight_split(s).splits > 1 ? "in parts" : "whole");
        }
    }
    printf("end\n");
}
int main(void) {
    int planes;
    long long rows;
    SvoxGatedFfn s{};
    while (scanf("%%d %%lld %%d %%d %%d", &planes, &rows, &s.dim, &s.hidden, &s.out) == 5) {
        s.rows = rows;
        if (planes == 1) say<1>(s);
        else say<3>(s);
    }
    return 0;
}
"""


def compiled(folder):
    """The program, in `folder`."""
    source, program = os.path.join(folder, "rules.cpp"), os.path.join(folder, "rules")
    with open(source, "w") as f:
        f.write(PROGRAM % SOURCE)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-o", program, source], check=True)
    return program


def kernels_of(program, planes, sizes):
    """For every (rows, features, hidden units, numbers of the result) of `sizes` the set of kernels its calls run on."""
    lines = "\n".join(f"{planes} {' '.join(map(str, size))}" for size in sizes)
    out = subprocess.run([program], input=lines, stdout=subprocess.PIPE, text=True, check=True).stdout
    return [set(part.strip().split("\n")) for part in out.split("end\n")[:-1]]


# Sizes on which every kernel runs, in both passes: rows, features, hidden units, numbers of the result; whole numbers of little.
NARROW = [(17, 33, 9), (32, 40, 49), (28, 130, 100), (49, 96, 28), (64, 100, 64), (60, 33, 127), (100, 40, 4), (76, 203, 49), (128, 72, 128)]
SIZES = ([(1, 40, 72, 24), (27, 100, 257, 30), (50, 33, 130, 65), (1500, 300, 100, 30), (1111, 20, 40, 77)]
         + [(rows, *widths) for rows in (9007, 98351) for widths in NARROW]
         + [(303, 700, 2048, 65), (303, 1024, 2048, 511), (2200, 150, 60, 24), (2101, 264, 203, 300), (4105, 1024, 3000, 1024), (9001, 130, 300, 200),
            (9011, 80, 33, 100), (12503, 136, 264, 264), (12503, 200, 513, 129), (16501, 129, 300, 513), (40003, 129, 300, 129), (40003, 300, 64, 20),
            (65603, 17, 40, 200)])
