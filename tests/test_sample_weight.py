"""The integer weight of a logit (csrc/sample_weight.h), compiled for the CPU: the same number whether the
compiler may fuse products and sums around it or not, and the weight that the sampler's definition asks for."""
import os
import subprocess

import numpy as np
import pytest

from llambda_amd import build

PROGRAM = r"""
#include "sample_weight.h"
#include <cstdio>
#include <vector>
int main(int, char** argv) {
  const long n = atol(argv[1]);
  std::vector<double> powers(llhip::kBatchBins), sharpness(n);
  std::vector<float> v(n), top(n);
  FILE* in = fopen(argv[2], "rb");
  bool ok = in && fread(powers.data(), 8, powers.size(), in) == powers.size();
  ok = ok && fread(sharpness.data(), 8, n, in) == (size_t)n && fread(v.data(), 4, n, in) == (size_t)n &&
       fread(top.data(), 4, n, in) == (size_t)n;
  if (!ok) return 1;
  for (long i = 0; i < n; ++i) {
    const llhip::Weighed w = llhip::weigh(powers.data(), v[i], top[i], sharpness[i]);
    const uint64_t out[2] = {(uint64_t)w.bin, w.weight};
    fwrite(out, 8, 2, stdout);
  }
}
"""
BINS, ONE = 2048, 2.0 ** 44


@pytest.fixture(scope="module")
def weights(tmp_path_factory):
    """{contraction: (bins, weights)} of the same logits."""
    at = tmp_path_factory.mktemp("weights")
    (at / "weights.hip").write_text(PROGRAM)
    rng = np.random.default_rng(1)
    n = 400000
    temperature = np.exp(rng.uniform(-3, 3, size=n)).astype(np.float32).astype(np.float64)
    top = (rng.normal(size=n) * 10).astype(np.float32)
    below = rng.uniform(0, 34, size=n) * temperature
    v = (top - below).astype(np.float32)
    v[:1000] = top[:1000]
    powers = np.exp(-np.arange(BINS) / 64) * ONE
    sharpness = 1 / temperature
    (at / "in").write_bytes(powers.tobytes() + sharpness.tobytes() + v.tobytes() + top.tobytes())
    got = {}
    for mode in ("off", "on", "fast-honor-pragmas"):
        program = str(at / f"weights_{mode}")
        subprocess.run([build.HIPCC, "-x", "hip", "--cuda-host-only", "-O3", "-std=c++20", "-march=native",
                        f"-ffp-contract={mode}", "-I", build.CSRC, str(at / "weights.hip"), "-o", program],
                       check=True, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)
        out = subprocess.run([program, str(n), str(at / "in")], check=True, stdout=subprocess.PIPE).stdout
        got[mode] = np.frombuffer(out, np.uint64).reshape(n, 2)
    x = (top.astype(np.float64) - v.astype(np.float64)) * sharpness
    return got, x


@pytest.mark.skipif(not os.path.exists(build.HIPCC), reason="no hipcc here")
def test_the_same_integer_under_every_contraction(weights):
    got, _ = weights
    for mode in ("on", "fast-honor-pragmas"):
        differ = (got[mode] != got["off"]).any(1)
        assert not differ.any(), f"{mode}: {differ.sum()} weights differ"


@pytest.mark.skipif(not os.path.exists(build.HIPCC), reason="no hipcc here")
def test_weights_are_the_exponentials(weights):
    """To 2e-9 of themselves and half a step of 2^-44; bins ascend with the distance from the highest."""
    got, x = weights
    bins, w = got["off"][:, 0].astype(np.int64), got["off"][:, 1].astype(np.float64) / ONE
    inside = 64 * x < BINS - 1 - 1e-6
    assert inside.sum() > 1000 and (~inside).sum() > 1000
    assert np.all(np.abs(bins[inside] - np.floor(64 * x[inside])) <= 1)  # (a border may round either way)
    want = np.exp(-x)
    assert np.all(np.abs(w - want)[inside] <= 2e-9 * want[inside] + 2.0 ** -45)
    outside = 64 * x >= BINS - 1 + 1e-6
    assert np.all(bins[outside] == BINS - 1) and not w[outside].any()
    assert np.all(w[x == 0] == 1) and (x == 0).sum() >= 1000
