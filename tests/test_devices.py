"""Calls of a context whose device is not the current one: their stream is that of the context's device, and the current device stays."""
import os
import subprocess
import tempfile
from types import SimpleNamespace

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


class _Rows:
    """Stands in for a CUDA tensor."""
    is_cuda = True

    def __init__(self, dtype, *shape):
        self.dtype, self.shape, self.device = dtype, shape, "cuda:0"

    def dim(self):
        return len(self.shape)

    def is_contiguous(self):
        return True

    def data_ptr(self):
        return 16

    def new_empty(self, *shape, dtype=None):
        return _Rows(dtype or self.dtype, *(shape[0] if isinstance(shape[0], tuple) else shape))


def test_every_call_goes_to_the_stream_of_its_context(monkeypatch):
    import torch

    from makepad_b200 import _lib, quant_linear as ql
    raw = {0: 1000, 1: 2000}
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", raw.__getitem__, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 1, raising=False)
    monkeypatch.setattr(torch, "empty", lambda *a, **k: _Rows(torch.float32, 1, 1))
    streams = []

    class Lib:
        def __getattr__(self, name):
            return lambda *a: streams.append((name, a[-1])) or 0
    ctx = SimpleNamespace(h=None, device=0, lib=Lib(), check=lambda st: None)

    def linear(fmt):
        return ql.QuantLinear(SimpleNamespace(ctx=ctx, h=None, fmt=fmt, N=64, K=32))
    f32, u8 = torch.float32, torch.uint8
    linear(_lib.FMT_Q4)(_Rows(f32, 2, 32))
    linear(_lib.FMT_Q4).forward_swiglu(_Rows(f32, 2, 64))
    linear(_lib.FMT_NVFP4)((_Rows(u8, 2, 16), _Rows(u8, 2, 2), 1.0))
    ql.nvfp4_quantize(ctx, _Rows(f32, 2, 32))
    ql.nvfp4_quantize(ctx, _Rows(f32, 2, 64), swiglu_fused=True)
    ql.swiglu(ctx, _Rows(f32, 2, 64))
    assert [n for n, _ in streams] == ["mpq_q4_linear_forward", "mpq_q4_linear_forward_swiglu", "mpq_nvfp4_gemm_forward", "mpq_nvfp4_quantize_activations",
                                       "mpq_nvfp4_quantize_swiglu", "mpq_swiglu"]
    assert {s for _, s in streams} == {1000}


PROGRAM = r"""
#include "on_device.h"
#include <cstdio>
static int current = 0, sets = 0, fails = 0;
extern "C" cudaError_t cudaGetDevice(int* d) { *d = current; return fails == 1 ? cudaErrorUnknown : cudaSuccess; }
extern "C" cudaError_t cudaSetDevice(int d) { ++sets; if (fails == 2) return cudaErrorUnknown; current = d; return cudaSuccess; }
using namespace mpq;
int main()
{
    int bad = 0;
    { current = 3; sets = 0; const OnDevice on(1); bad += on.error != cudaSuccess || current != 1; }
    bad += current != 3 || sets != 2;
    { sets = 0; const OnDevice on(3); bad += on.error != cudaSuccess || current != 3; }
    bad += current != 3 || sets != 0;
    { sets = 0; fails = 1; const OnDevice on(1); bad += on.error == cudaSuccess; }
    bad += current != 3 || sets != 0;
    { sets = 0; fails = 2; const OnDevice on(1); bad += on.error == cudaSuccess; }
    bad += current != 3 || sets != 1;
    std::printf("%d\n", bad);
    return bad;
}
"""


def test_the_current_device_comes_back():
    with tempfile.TemporaryDirectory() as tmp:
        src, exe = os.path.join(tmp, "t.cpp"), os.path.join(tmp, "t")
        open(src, "w").write(PROGRAM)
        subprocess.check_call(["g++", "-std=c++17", "-O1", "-Wall", "-I", os.path.join(ROOT, "makepad_b200", "csrc"), "-I", "/usr/local/cuda/include", src, "-o", exe])
        out = subprocess.run([exe], capture_output=True, text=True)
        assert out.returncode == 0 and out.stdout.strip() == "0", out.stdout + out.stderr


@pytest.mark.parametrize("call", ["q4_linear_forward", "q4_linear_forward_static", "q4_linear_forward_allreduce", "swiglu", "q4_linear_forward_swiglu", "nvfp4_gemm_forward", "nvfp4_quantize_activations", "nvfp4_quantize_swiglu", "residual_norm", "kv_plan",
                                  "kv_append", "paged_attention", "prompt_attention"])
def test_forward_calls_leave_the_current_device(call):
    """Each of them, or what it calls, holds an OnDevice and sets no device itself."""
    for f in ("mpq.cu", "block.cu"):
        text = open(os.path.join(ROOT, "makepad_b200", "csrc", f)).read()
        at = text.find(f'extern "C" int32_t mpq_{call}(')
        if at >= 0:
            body = text[at:text.index("\n}\n", at)]
            if "attention_launch(" in body:
                at = text.index("static int32_t attention_launch(")
                body = text[at:text.index("\n}\n", at)]
            assert "OnDevice on(ctx->device);" in body and "cudaSetDevice" not in body
            return
    raise AssertionError(call)


@pytest.mark.gpu
def test_a_thread_that_has_made_no_call_yet(ctx):
    """A host thread's first call of CUDA is one of the library's."""
    import threading

    import makepad_b200 as m
    import torch
    from makepad_b200 import synth
    lin = m.QuantLinear(m.Q4Weight(ctx, *synth.q4_weight(256, 512, seed=0)))
    x = torch.randn(3, 512, device="cuda")
    want, got, rows = lin(x), torch.empty(3, 256, device="cuda"), torch.empty(3, 512, device="cuda")
    torch.cuda.synchronize()
    status = []

    def work():
        status.append(ctx.lib.mpq_residual_norm(ctx.h, x.data_ptr(), 0, 3, 512, None, rows.data_ptr(), None, None, 0, 1.0, None, 1e-6, None, 0, None))
        status.append(ctx.lib.mpq_q4_linear_forward(ctx.h, lin.w.h, rows.data_ptr(), 3, got.data_ptr(), None))
    t = threading.Thread(target=work)
    t.start()
    t.join()
    torch.cuda.synchronize()
    assert status == [0, 0] and torch.equal(got, want)
