"""The powers of two that the attention of many rows makes by multiplications and additions, by themselves."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include "attention_many.cuh"
__global__ void powers(const float* x, float* y, long long pairs)
{
    const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= pairs) return;
    const uint64_t v = mpq::power2(mpq::pair_of(x[2 * i], x[2 * i + 1]));
    y[2 * i] = __uint_as_float((uint32_t)v);
    y[2 * i + 1] = __uint_as_float((uint32_t)(v >> 32));
}
extern "C" int run(const float* x, float* y, long long pairs)
{
    powers<<<(unsigned)((pairs + 255) / 256), 256>>>(x, y, pairs);
    const cudaError_t e = cudaGetLastError();
    return e != cudaSuccess ? (int)e : (int)cudaDeviceSynchronize();
}
"""


@pytest.fixture(scope="module")
def powers(tmp_path_factory):
    import torch
    at = tmp_path_factory.mktemp("powers")
    (at / "p.cu").write_text(PROGRAM)
    subprocess.check_call([os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc"), "-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-std=c++17", "--expt-relaxed-constexpr", "-Xcompiler", "-fPIC",
                           "-shared", "-I", os.path.join(ROOT, "makepad_b200", "csrc"), str(at / "p.cu"), "-o", str(at / "p.so")])
    lib = C.CDLL(str(at / "p.so"))
    lib.run.argtypes = [C.c_void_p, C.c_void_p, C.c_longlong]

    def run(x):
        assert x.size % 2 == 0
        x = torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)).cuda()
        y = torch.empty_like(x)
        torch.cuda.synchronize()
        assert lib.run(x.data_ptr(), y.data_ptr(), x.numel() // 2) == 0
        return y.cpu().numpy().astype(np.float64)
    return run


# a cubic is within 7.5e-5 of 2^f where |f| <= 1/2 (relative); f is exact, three roundings of fp32 in the cubic, and the exponent is added exactly
NEAR = 7.5e-5 + 4 * 2.0 ** -24


def test_powers_over_their_range(powers):
    rng = np.random.default_rng(1)
    whole = np.arange(-125, 9)
    x = np.concatenate([rng.uniform(-125.5, 8, 1 << 20), whole, np.repeat(whole, 2000) + np.tile(np.linspace(-0.5, 0.5, 2000), whole.size), np.linspace(-1, 1, 1 << 16),
                        np.nextafter(whole + 0.5, 99, dtype=np.float32), np.nextafter(whole + 0.5, -99, dtype=np.float32)]).astype(np.float32)
    x = x[(x <= 8) & (x >= -125.5)]
    x = x[:x.size // 2 * 2]
    want = np.exp2(x.astype(np.float64))
    off = np.abs(powers(x) - want) / want
    assert off.max() <= NEAR, (off.max(), x[off.argmax()])
    # (the bound is met: it is this cubic that was measured, not an exact power)
    assert off.max() >= 7e-5


def test_powers_at_and_below_the_smallest(powers):
    """Down to -126 the value may lie a little below 2^-126, where a step is 2^-149; everything below gives what -126 gives."""
    x = np.linspace(-126, -125.5, 1 << 14).astype(np.float32)
    want = np.exp2(x.astype(np.float64))
    # the smallest: 0.99993 of 2^-126 without the bit in front of its fraction is 0.99986 of it
    assert (np.abs(powers(x) - want) <= 2 * NEAR * want).all()
    low = np.array([-126, -126.00001, -127, -149, -1000, -3e38, -np.inf, -1e30], dtype=np.float32)
    y = powers(low)
    assert (y == y[0]).all() and abs(y[0] - 2.0 ** -126) <= 2 * NEAR * 2.0 ** -126


def test_powers_of_a_pair_do_not_mix(powers):
    a, b = np.float32(-100.3), np.float32(7.7)
    both = powers(np.array([a, b, b, a, a, a, b, b], dtype=np.float32))
    assert both[0] == both[3] == both[4] == both[5] and both[1] == both[2] == both[6] == both[7]
