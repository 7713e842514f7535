"""The serving operators' refusals, on the CPU: bad calls are turned down before any launch."""

from __future__ import annotations

import subprocess
import sys

import pytest
import torch

from conftest import PKG_PARENT
from tkmi import _lib, ops

S3 = _lib.strides([64, 64, 64])
S2 = _lib.strides([64, 64])
S4 = _lib.strides([64, 64, 64, 64])


def _window(dtype=1, b=1, h=4, hkv=2, sq=8, sk=8, hd=64, scale=0.1, window=4, sinks=0, q=16, k=16, strides=S3, kv=None,
            kvs=0, invariant=0, ws=None, size=0):
    return _lib.load().tk_window_attn(q, S3, k, strides, 16, S3, 16, S3, dtype, b, h, hkv, sq, sk, hd, scale, window,
                                      sinks, kv, kvs, invariant, ws, size, None)


@pytest.mark.parametrize("call,code", [
    (dict(dtype=0), -1), (dict(dtype=3), -1), (dict(h=3), -1), (dict(sq=9), -1), (dict(window=0), -1),
    (dict(sinks=-1), -1), (dict(scale=0.0), -1), (dict(scale=float("nan")), -1), (dict(scale=float("inf")), -1),
    (dict(hd=12), -2), (dict(hd=264), -2), (dict(q=None), -1), (dict(k=24), -2), (dict(b=-1), -1),
    (dict(strides=_lib.strides([64, 64, 60])), -2), (dict(kv=16, kvs=7), -1), (dict(sk=1 << 30), -1),
    (dict(sk=100000, window=100000), -1),  # splits its keys and has no workspace
    (dict(sk=100000, window=100000, ws=8, size=1 << 30), -1), (dict(sk=100000, window=100000, ws=16, size=64), -1),
    (dict(b=0), 0), (dict(sq=0), 0), (dict(h=0, hkv=0), 0),
])
def test_window_attention_refuses(call, code):
    assert _window(**call) == code
    assert code == 0 or _lib.load().tk_last_error_string().decode()


def _paged(dtype=1, b=2, h=4, hkv=2, hd=64, pages=8, ps=16, table=16, stride=4, width=4, lengths=16, most=64, scale=0.1,
           window=0, sinks=0, invariant=0, ws=None, size=0, q=16, k=16, strides=S3):
    return _lib.load().tk_paged_attn(q, S2, k, strides, 16, S3, 16, S2, dtype, b, h, hkv, hd, pages, ps, table, stride,
                                     width, lengths, most, scale, window, sinks, invariant, ws, size, None)


@pytest.mark.parametrize("call,code", [
    (dict(dtype=0), -1), (dict(h=5), -1), (dict(hd=20), -2), (dict(hd=320), -2), (dict(ps=8), -2), (dict(ps=48), -2),
    (dict(ps=2048), -2), (dict(stride=3), -1), (dict(table=None), -1), (dict(lengths=None), -1), (dict(scale=-1.0), -1),
    (dict(window=-1), -1), (dict(sinks=-2), -1), (dict(k=8), -2), (dict(k=None), -1), (dict(pages=-1), -1),
    (dict(strides=_lib.strides([4, 64, 64])), -2), (dict(most=-1), -1), (dict(width=1 << 26, stride=1 << 26), -1),
    (dict(most=1 << 20), -1),  # splits its keys and has no workspace
    (dict(most=1 << 20, ws=8, size=1 << 30), -1), (dict(most=1 << 20, ws=16, size=100), -1),
    (dict(b=0), 0), (dict(h=0, hkv=0), 0),
])
def test_paged_attention_refuses(call, code):
    assert _paged(**call) == code
    assert code == 0 or _lib.load().tk_last_error_string().decode()


def test_window_workspace():
    size = _lib.load().tk_window_attn_workspace
    assert size(1, 4, 4, 5, 100000, 64, 100000, 0, 1) == 0  # batch-invariant: no split
    assert size(64, 16, 4, 500, 500, 64, 100, 4, 0) == 0    # enough rows
    assert size(1, 4, 4, 5, 100, 64, 20, 0, 0) == 0         # few keys: one workgroup's waves share them
    assert size(1, 4, 4, 5, 100000, 64, 100000, 0, 0) % (4 * 5 * 66 * 4) == 0
    assert size(1, 4, 4, 5, 100000, 64, 100000, 0, 0) > size(1, 4, 4, 5, 100000, 64, 4000, 0, 0) > 0
    assert size(1, 4, 4, 5, 100000, 64, 1 << 60, 0, 0) == size(1, 4, 4, 5, 100000, 64, 100000, 0, 0)
    assert size(0, 4, 4, 5, 10, 64, 4, 0, 0) == 0 and size(1, 4, 4, 5, 4, 64, 4, 0, 0) == -1


def test_paged_workspace():
    size = _lib.load().tk_paged_attn_workspace
    assert size(0, 8, 8, 64, 100000, 0, 0, 0) == 0
    assert size(1, 8, 8, 64, 16, 0, 0, 0) == 0  # one split writes its results
    whole = size(1, 8, 8, 64, 100000, 0, 0, 0)  # O, max and sum per split and head, two ints per sequence
    assert whole > 8 and (whole - 8) % (8 * 66 * 4) == 0
    assert size(1, 8, 8, 64, 100000, 64, 4, 0) <= size(1, 8, 8, 64, 100000, 0, 0, 0)
    assert size(1, 8, 3, 64, 16, 0, 0, 0) == -1 and size(1, 8, 8, 36, 16, 0, 0, 0) == -2
    # batch-invariant splits: their number goes with the length alone
    assert size(2, 8, 8, 64, 5000, 0, 0, 1) == 2 * size(1, 8, 8, 64, 5000, 0, 0, 1)


def test_cache_calls_refuse():
    lib = _lib.load()

    def append(b=1, n=1, hkv=1, hd=64, pages=4, ps=16, k=16, strides=S3, table=16, lengths=16, width=4, stride=4):
        return lib.tk_cache_append(k, strides, 16, S3, 16, S3, 16, S3, b, n, hkv, hd, pages, ps, table, stride, width,
                                   lengths, None, None)

    for call, code in [(dict(hd=12), -2), (dict(ps=24), -2), (dict(k=None), -1), (dict(k=2), -2), (dict(n=-1), -1),
                       (dict(lengths=None), -1), (dict(table=None), -1), (dict(b=2, stride=3), -1),
                       (dict(strides=_lib.strides([64, 7, 64])), -2), (dict(n=0), 0), (dict(b=0), 0),
                       (dict(pages=0), 0)]:
        assert append(**call) == code, call

    def state(rows=2, width=4, stride=4, table=16, lengths=16, refs=16, pages=8, ps=16):
        return (table, stride, width, rows, lengths, refs, pages, ps)

    def reserve(new=16, status=16, ws=16, size=1 << 20, **kw):
        return lib.tk_cache_reserve(*state(**kw), new, status, ws, size, None)

    for call, code in [(dict(new=None), -1), (dict(status=None), -1), (dict(ws=None), -1), (dict(size=31), -1),
                       (dict(ps=0), -2), (dict(refs=None), -1), (dict(lengths=None), -1), (dict(stride=2), -1),
                       (dict(rows=-1), -1), (dict(pages=-1), -1)]:
        assert reserve(**call) == code, call

    def pages_args(k=16, layers=1, hkv=2, hd=64, strides=S4):
        return (k, strides, 16, S4, layers, hkv, hd)

    def fork(parents=16, children=16, n=1, status=16, ws=16, size=1 << 20, cache=pages_args(), **kw):
        return lib.tk_cache_fork(*cache, *state(**kw), parents, children, n, status, ws, size, None)

    for call, code in [(dict(parents=None), -1), (dict(n=-1), -1), (dict(status=None), -1), (dict(size=39), -1),
                       (dict(cache=pages_args(k=None)), -1), (dict(cache=pages_args(k=8)), -2),
                       (dict(cache=pages_args(hd=4)), -2), (dict(cache=pages_args(layers=-1)), -1),
                       (dict(cache=pages_args(strides=_lib.strides([1, 64, 64, 64]))), -2),
                       (dict(cache=pages_args(hkv=65535, hd=256), ps=1024), -1), (dict(width=-1), -1),
                       (dict(rows=(1 << 18) + 1, width=1, stride=1), -2)]:
        assert fork(**call) == code, call
    assert lib.tk_cache_free(*state(), None, 1, None) == -1
    assert lib.tk_cache_free(*state(), 16, -1, None) == -1
    assert lib.tk_cache_free(*state(), None, 0, None) == 0
    assert lib.tk_cache_compact(*pages_args(), *state(), None, 16, 1 << 20, None) == -1
    assert lib.tk_cache_compact(*pages_args(), *state(), 16, 16, 4 * 16, None) == -1
    assert lib.tk_cache_workspace(-1, 4, 0) == -1 and lib.tk_cache_workspace(2, 8, 3) >= 4 * (6 + 16)


@pytest.mark.parametrize("scale,code", [(2.3e38, 0), (2.36e38, -1), (3.0e38, -1), (-1.0, -1), (1e-45, 0)])
def test_scales_whose_log2_units_are_infinite_are_refused(scale, code):
    """Scores are scaled by scale * log2(e); an infinite factor would make a score of 0 NaN."""
    assert _window(b=0, scale=scale) == code and _paged(b=0, scale=scale) == code


def test_append_with_a_status_refuses():
    """As without one, and a status that is not there."""
    lib = _lib.load()

    def append(hd=64, ps=16, n=1, status=16, lengths=16):
        return lib.tk_cache_append_reserved(16, S3, 16, S3, 16, S3, 16, S3, 1, n, 1, hd, 4, ps, 16, 4, 4, lengths, None,
                                            status, None)

    for call, code in [(dict(status=None), -1), (dict(hd=12), -2), (dict(ps=24), -2), (dict(lengths=None), -1),
                       (dict(n=0), 0)]:
        assert append(**call) == code, call
        assert code == 0 or "tk_cache_append_reserved" in lib.tk_last_error_string().decode()


def test_launches_of_too_many_workgroups_are_refused():
    """A launch holds fewer than 2^32 threads: 2^24 workgroups of 256."""
    lib = _lib.load()
    state = (16, 4, 4, 1 << 18, 16, 16, 8, 16)
    assert _window(b=1 << 20, h=32, hkv=32) == -2
    assert _window(b=1 << 20, h=32, hkv=32, sq=300, sk=300) == -2
    assert _paged(b=1 << 23) == -2
    assert lib.tk_cache_append(16, S3, 16, S3, 16, S3, 16, S3, 1 << 14, 1 << 15, 1, 64, 4, 16, 16, 4, 4, 16, None,
                               None) == -2
    assert lib.tk_cache_fork(16, S4, 16, S4, 2, 2, 64, *state, 16, 16, 1 << 22, 16, 16, 1 << 40, None) == -2
    assert lib.tk_cache_free(*state, 16, 1 << 24, None) == -1


def test_a_join_of_too_many_workgroups_is_refused_before_the_first_launch():
    """2^22 workgroups attend, but 2^24 would join them: the refusal (and not what a launch says here)."""
    call = dict(b=65536, h=32, hkv=32, hd=128, pages=8, ps=16, width=128, stride=128, most=2048, invariant=1, ws=16)
    need = _lib.load().tk_paged_attn_workspace(65536, 32, 32, 128, 2048, 0, 0, 1)
    assert need > 0 and _paged(**call, size=need - 1) in (-1, -2)
    assert _paged(**call, size=need) == -2
    assert "too many workgroups" in _lib.load().tk_last_error_string().decode()


def test_import_needs_no_gpu_build_of_torch():
    """A torch without a GPU backend has no current raw stream: the package imports, its operators say what they need."""
    code = ("import torch, sys\n"
            "del torch._C._cuda_getCurrentRawStream\n"
            "sys.path.insert(0, %r)\n"
            "import tkmi\n"
            "v = torch.zeros(1, dtype=torch.int32)\n"
            "try: tkmi.ops.cache_free(v[None], v, v, v, 16)\n"
            "except RuntimeError as e: assert 'GPU only' in str(e)\n"
            "else: raise SystemExit(2)\n") % str(PKG_PARENT)
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr[-500:]


def test_wrappers_refuse_on_the_cpu():
    half = torch.zeros(1, 2, 4, 64, dtype=torch.float16)
    table, vec = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.window_attention(half, half, half, 0.1, 4)
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.paged_attention(half[:, :, 0], half, half, table, vec, 0.1)
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.cache_append(half, half, half, half, table, vec)
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.cache_reserve(table, vec, vec, vec, 16)
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.cache_free(table, vec, vec, vec, 16)
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.cache_fork(half, half, table, vec, vec, vec, vec)
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.cache_compact(half, half, table, vec, vec)
    with pytest.raises(TypeError, match="int32"):
        ops.cache_reserve(table.long(), vec, vec, vec, 16)


def test_serving_kernels_use_no_scratch():
    """A spilled accumulator costs several times a kernel's time and no result shows it."""
    import json

    from tkmi import build as tkbuild

    if not tkbuild.RESOURCE_PATH.exists():
        pytest.skip("library not built")
    usage = json.loads(tkbuild.RESOURCE_PATH.read_text())
    # types x head-dim tiles x (one or a few workgroups per sequence; masked or not), the joins, the cache's
    expected = {"paged_attn_kernel": 16, "window_attn_kernel": 16, "window_split_kernel": 16, "split_join_kernel": 4,
                "cache_": 7}
    for name, least in expected.items():
        found = {k: v["scratch"] for k, v in usage.items() if name in k}
        assert len(found) >= least, (name, len(found))
        assert not any(found.values()), found
