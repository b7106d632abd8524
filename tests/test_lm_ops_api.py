"""The operators around the scan layers without a GPU: argument checks of the C
ABI answer before any launch, and the Python calls refuse CPU tensors instead
of falling back."""
import ctypes

import pytest
import torch

P = ctypes.c_void_p(4096)  # never dereferenced: validation fails first


@pytest.fixture(scope="module")
def lib():
    from mamba import _native

    return _native.load()


def _says(lib, status, text):
    assert status == 1
    assert text in lib.mamba_ss_last_error()


def test_norm_arguments(lib):
    fwd = lambda dt=0, rows=4, dim=8, x=P, res=None, h=None: lib.mamba_ss_rms_norm_fwd(  # noqa: E731
        None, dt, 0, rows, dim, 1e-5, x, dim, res, dim, P, P, h)
    _says(lib, fwd(dt=5), b"data types")
    _says(lib, fwd(rows=0), b"rows")
    _says(lib, fwd(dim=16385), b"dim")
    _says(lib, fwd(x=None), b"non-null")
    _says(lib, fwd(res=P), b"non-null")
    _says(lib, fwd(h=P), b"non-null")
    st = lib.mamba_ss_rms_norm_fp8(None, 0, 0, 4, 100, 1e-5, P, 100, None, 0, P, P, 100, P, 1, None)
    _says(lib, st, b"multiple of 16")
    assert lib.mamba_ss_rms_norm_bwd_workspace_bytes(0, 8) == 0
    need = lib.mamba_ss_rms_norm_bwd_workspace_bytes(1000, 768)
    assert need >= 768 * 4 and need % (768 * 4) == 0
    bwd = lambda ws, dres=None, dt=1: lib.mamba_ss_rms_norm_bwd(  # noqa: E731
        None, dt, 1, 0, 1000, 768, 1e-5, P, 768, P, 768, None, 0, P, P, dres, P, P, ws)
    _says(lib, bwd(need - 1, P), b"workspace needs")
    _says(lib, bwd(need), b"dresidual")
    _says(lib, bwd(need, P, dt=0), b"dresidual")


def test_fp8_arguments(lib):
    q = lambda dt=0, cm=0, b=2, l=3, k=40, stride=48, codes=P, ss=1: lib.mamba_ss_quantize_fp8(  # noqa: E731
        None, dt, cm, b, l, k, P, k, codes, stride, P, ss)
    _says(lib, q(dt=3), b"x_dtype")
    _says(lib, q(k=0), b"positive")
    _says(lib, q(stride=40), b"multiple of 16")
    _says(lib, q(stride=32), b"multiple of 16")
    _says(lib, q(codes=ctypes.c_void_p(4097)), b"16-byte")
    _says(lib, q(codes=None), b"non-null")
    _says(lib, q(cm=1, b=70000), b"too large")
    _says(lib, q(k=140, stride=144, ss=1), b"cover the row")
    st = lib.mamba_ss_dequantize_fp8(None, 0, 2, 40, P, 48, P, 1, ctypes.c_void_p(4100))
    _says(lib, st, b"16-byte")
    mm = lambda dt=1, tr=0, m=4, n=4, z=1, k=64, sa=64, a=P: lib.mamba_ss_fp8_matmul(  # noqa: E731
        None, dt, tr, m, n, z, k, a, sa, P, 1, P, 64, P, 1, P)
    _says(lib, mm(dt=2), b"out_dtype")
    _says(lib, mm(m=0), b"positive")
    _says(lib, mm(tr=1, z=2), b"one batch")
    _says(lib, mm(sa=72), b"multiple of 16")
    _says(lib, mm(a=None), b"non-null")
    _says(lib, mm(m=2 ** 31 - 1, n=2 ** 31 - 1), b"too large")


def test_sample_arguments(lib):
    s = lambda dt=0, rows=2, vocab=10, z=P, u=P: lib.mamba_ss_sample_tokens(  # noqa: E731
        None, dt, rows, vocab, z, vocab, u, None, None, None, None, 1.0, 0, 1.0, 0.0, P)
    _says(lib, s(dt=9), b"dtype")
    _says(lib, s(rows=0), b"rows")
    _says(lib, s(vocab=360449), b"vocab")
    _says(lib, s(z=None), b"non-null")
    _says(lib, s(u=None), b"non-null")


def test_no_fallback_on_cpu_tensors():
    import mamba

    x, w = torch.randn(4, 32), torch.ones(32)
    for call in (lambda: mamba.rms_norm_fn(x, w), lambda: mamba.rms_norm_fp8(x, w),
                 lambda: mamba.quantize_fp8(x), lambda: mamba.fp8_linear(x, x),
                 lambda: mamba.dequantize_fp8(x.to(torch.float8_e4m3fn),
                                              torch.ones(4, 1).to(torch.float8_e8m0fnu)),
                 lambda: mamba.sample_tokens(x, torch.rand(4))):
        with pytest.raises(ValueError, match="CUDA"):
            call()


@pytest.mark.timeout(900)
def test_library_builds_without_torch():
    """The C library serves callers that have no PyTorch; only the operators' PyTorch
    host side needs it."""
    import subprocess
    import sys
    from pathlib import Path

    build = Path(__file__).resolve().parents[1] / "jax-mambas_b200" / "build.py"
    code = ("import runpy, sys; sys.modules['torch'] = None; sys.argv = ['build.py']; "
            f"runpy.run_path({str(build)!r}, run_name='__main__')")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    assert "libmamba_ss_b200.so" in r.stdout and "_mamba_ops.so not built" in r.stdout


def test_missing_binding_says_how_to_build_it(lib, monkeypatch, tmp_path):
    from mamba import _native, _ops

    monkeypatch.setattr(_ops, "_OPS", None)
    monkeypatch.setattr(_native, "_PKG_ROOT", tmp_path)
    with pytest.raises(FileNotFoundError, match="build.py"):
        _ops.ops()


def test_row_counts_that_pass_64_bits_are_refused(lib):
    """2^40 rows of 2^23 blocks are 2^63: no number of 64 bits with a sign."""
    st = lib.mamba_ss_quantize_fp8(None, 0, 0, 1 << 20, 1 << 20, 1 << 30, P, 1 << 30, P, 1 << 30,
                                   P, 1 << 23)
    _says(lib, st, b"too large")
