"""A request's rows from a list of offsets that lies on the device, where nothing can be refused: whatever stands there, they are rows that
there are.  The rule is the kernels' own code, compiled for the host."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "biv_b200", "csrc")


def test_rows_of_any_two_offsets(tmp_path):
    src, exe = tmp_path / "rows.cpp", str(tmp_path / "rows")
    src.write_text(r"""
#include <climits>
#include <cstdio>
#include <random>
#include "rows_of.h"
using namespace bivmoe;
static int check(int from, int to, int n_tokens) {
    auto kept = [&](long long x) { return x < 0 ? 0 : x > n_tokens ? (long long)n_tokens : x; };
    const long long a = kept(from), b = kept(to);
    const RowsOf r = rows_of(from, to, n_tokens);
    if (r.first == a && r.n == (b > a ? b - a : 0) && r.n >= 0 && (long long)r.first + r.n <= n_tokens) return 0;
    printf("%d %d %d: %d %d\n", from, to, n_tokens, r.first, r.n);
    return 1;
}
int main() {
    const int ends[] = {INT_MIN, INT_MIN + 1, -130, -7, -1, 0, 1, 20, 90, 130, 131, 1 << 30, INT_MAX - 1, INT_MAX};
    for (int n : {0, 1, 130, 1 << 30, INT_MAX})
        for (int from : ends)
            for (int to : ends)
                if (check(from, to, n)) return 1;
    std::mt19937 rng(1);
    for (int i = 0; i < 1000000; i++)
        if (check((int)rng(), (int)rng(), (int)(rng() >> (1 + rng() % 31)))) return 1;
    return 0;
}
""")
    # -ftrapv: a sum or difference that overflows ends the program
    subprocess.run(["g++", "-std=c++17", "-O1", "-ftrapv", "-Wall", "-Werror", "-I", CSRC, "-o", exe, str(src)], check=True)
    r = subprocess.run([exe], timeout=60, capture_output=True, text=True)
    assert r.returncode == 0, r.stdout


def test_offsets_are_read_by_that_rule_alone():
    for name, of in (("linear.cuh", "c"), ("linear_tc.cuh", "c"), ("verify.cu", "a")):
        with open(os.path.join(CSRC, name)) as f:
            lines = [line.split("//")[0] for line in f]
        reads = [line for line in lines if f"{of}.first[" in line]
        assert reads and all("rows_of(" in line for line in reads), (name, reads)
