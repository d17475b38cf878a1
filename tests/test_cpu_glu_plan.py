"""The gated projection's plan and workspace size (csrc/glu_plan.h) on the host,
for every number of SM pairs that a device, or a share of one, can offer."""
import ctypes as C
import os
import random
import subprocess

import pytest

from conftest import ROOT

CSRC = os.path.join(ROOT, "embeddinggemma2-amdkfd_b200", "csrc")
PAIRS, MOST = 74, 8
SHIM = """
#include "glu_plan.h"
extern "C" {
void plan(unsigned n, unsigned k, unsigned m, int dx, int w, int pairs, int most, int *out) {
    const eg2::GluPlan p = eg2::glu_plan(n, k, m, dx != 0, w, pairs, most);
    out[0] = p.splits, out[1] = p.dxc;
}
int most_splits(unsigned n, unsigned k, unsigned m) { return eg2::glu_most_splits(n, k, m); }
unsigned long long bytes(unsigned n, unsigned k, unsigned m, int splits) { return eg2::glu_grad_bytes(n, k, m, splits); }
}
"""


@pytest.fixture(scope="module")
def H(tmp_path_factory):
    d = tmp_path_factory.mktemp("plan")
    (d / "shim.cpp").write_text(SHIM)
    so = str(d / "plan.so")
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-shared", "-fPIC", "-I", CSRC, str(d / "shim.cpp"), "-o", so],
                   check=True)
    lib = C.CDLL(so)
    lib.bytes.restype = C.c_ulonglong

    def plan(n, k, m, dx, w, pairs, most):
        out = (C.c_int * 2)()
        lib.plan(n, k, m, dx, w, pairs, most, out)
        return out[0], out[1]

    lib.plan_of = plan
    return lib


def shapes(count):
    rng = random.Random(7)
    size = lambda most: 8 * round(2 ** rng.uniform(0, most))
    return [(round(2 ** rng.uniform(0, 15)), size(9), size(11)) for _ in range(count)] + \
        [(4096, 512, 2048), (3930, 2264, 6584), (1, 8, 8), (2048, 512, 2048)]


def test_parts_never_pass_the_workspace(H, eg2):
    size = eg2._lib.load().eg2_glu_grad_workspace
    for n, k, m in shapes(40):
        most = H.most_splits(n, k, m)
        assert size(n, k, m) == H.bytes(n, k, m, most)
        for pairs in range(1, PAIRS + 1):
            for w in (0, 1, 2):
                splits, dxc = H.plan_of(n, k, m, 1, w, pairs, most)
                assert 1 <= splits <= most
                # Every kind of tile has a cluster: dx's own and the weights' own, or all clusters both.
                assert dxc == -1 and w if dxc < 0 else 1 <= dxc <= pairs - (1 if w else 0), (n, k, m, pairs, w)
                assert H.bytes(n, k, m, splits) <= size(n, k, m)
        for w in (1, 2):
            assert H.plan_of(n, k, m, 0, w, PAIRS, most) == (1, 0)


def test_a_share_of_the_device_can_want_more_parts(H):
    """The bound matters: without it these plans take more parts than are sized."""
    for n, k, m, pairs in ((4096, 512, 2048, 60), (3930, 2264, 6584, 72)):
        most = H.most_splits(n, k, m)
        assert max(H.plan_of(n, k, m, 1, w, pairs, MOST)[0] for w in (0, 1, 2)) > most


def test_the_whole_device_plans_without_the_bound(H):
    for n, k, m in shapes(200):
        most = H.most_splits(n, k, m)
        for w in (0, 1, 2):
            assert H.plan_of(n, k, m, 1, w, PAIRS, most) == H.plan_of(n, k, m, 1, w, PAIRS, MOST)


def test_few_elements_keep_their_rests(H, eg2):
    """With few elements in the inner gradients or in dx the workspace has both parts of the former."""
    half = lambda n, m: (2 * n * m + 255) // 256 * 256
    for n, k, m, parts in ((1, 2048, 8, 4), (1, 2048, 6136, 4), (1, 2048, 6144, 2), (1, 1016, 8192, 4),
                           (1, 1024, 8192, 2), (767, 64, 8, 4), (768, 64, 8, 2), (95, 64, 64, 4), (96, 64, 64, 2),
                           (127, 8, 4096, 4), (128, 8, 4096, 2)):
        assert H.bytes(n, k, m, 1) == parts * half(n, m)
        assert eg2._lib.load().eg2_glu_grad_workspace(n, k, m) >= parts * half(n, m)
