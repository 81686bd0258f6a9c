"""The rule that cuts a product of codes (q8_plan in qw_gemm_q8.cu), compiled from the library's source for the host: which forms
it reaches at all, that the shapes of the GPU tests reach each of them, and that rings and sums fit what a launch asks for."""
import os
import re
import subprocess

import pytest

from tests.test_gpu_linear_q8_forms import SHAPES

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

MAIN = r"""
int main() {
    int t, n, k;
    while (scanf("%d %d %d", &t, &n, &k) == 3) {
        const Q8Plan p = q8_plan(n, t, k, 148);
        const int nkb = (k + kBK - 1) / kBK;
        const long long tiles = (long long)((n + p.ctas * kBM - 1) / (p.ctas * kBM)) * ((t + p.bn - 1) / p.bn);
        const int s = p.nsplit ? split_stages(p, (nkb + p.nsplit - 1) / p.nsplit, q8_alone(p, tiles)) : 0;
        printf("%d %d %d %d %d %lld\n", p.ctas, p.bn, p.nsplit, s, s * split_stage_bytes(p.ctas, p.bn), tiles);
    }
}
"""


@pytest.fixture(scope="module")
def plans(tmp_path_factory):
    with open(os.path.join(ROOT, "common_b200", "csrc", "qw_gemm_q8.cu")) as f:
        s = f.read()
    cut = lambda a, b: s[s.index(a) : s.index(b, s.index(a))]  # noqa: E731
    constants = re.findall(r"^constexpr int (?:kBM|kClusterMax|kPairBM) = .*$", s, re.M)
    text = "#include <initializer_list>\n#include <math.h>\n#include <stdio.h>\n#define __host__\n#define __device__\n" + "\n".join(constants) + "\n" + \
        cut("__host__ __device__ constexpr int split_stage_bytes", "template <int CTAS, int BN, int EPI>") + \
        cut("struct Q8Plan {", "template <int EPI>\nconst void *q8_kernel") + \
        cut("constexpr Q8Plan kForms", "// Every kernel opted in") + cut("float q8_cost(", "cudaError_t q8_gemm_launch") + MAIN
    tmp = tmp_path_factory.mktemp("plan")
    (tmp / "plan.cpp").write_text(text)
    exe = str(tmp / "plan")
    subprocess.run(["/usr/bin/g++", "-std=c++17", "-O2", "-ffp-contract=off", str(tmp / "plan.cpp"), "-o", exe], check=True)

    def ask(shapes):
        r = subprocess.run([exe], input="\n".join("%d %d %d" % s for s in shapes), capture_output=True, text=True, check=True)
        return [tuple(map(int, line.split())) for line in r.stdout.splitlines()]
    return ask


def many():
    """Shapes over the whole range, ragged and whole."""
    steps = lambda lo, hi, n: sorted({int(round(lo * (hi / lo) ** (i / (n - 1)))) for i in range(n)})  # noqa: E731
    tokens = sorted(set(steps(1, 20000, 60)) | {16, 32, 64, 128, 256, 512, 1024, 4096, 8192})
    features = sorted(set(steps(1, 40000, 45)) | {1152, 4096, 6144, 24576})
    codes = sorted(set(steps(1, 131071, 45)) | {896, 4096, 12288})
    return [(t, n, k) for t in tokens for n in features for k in codes]


def test_every_form_is_tested(plans):
    reached = {p[:3] for p in plans(many())}
    assert len(reached) == 27
    assert {p[:3] for p in plans(SHAPES)} == reached


def test_rings_fit(plans):
    """Shared memory of a CTA, the sums of a tile in it, ranges that are not empty, clusters of at most eight CTAs."""
    shapes = many()
    for (t, n, k), (ctas, bn, nsplit, stages, room, _) in zip(shapes, plans(shapes)):
        if nsplit == 0:
            continue
        assert 1 <= stages <= 12 and room <= 200 * 1024 and nsplit <= -(-k // 128) and nsplit * ctas <= 8
        assert nsplit == 1 or room >= bn * 128 * 4
