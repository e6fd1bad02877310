"""Rotary positions, KV append and sampling without a GPU: argument checks before any CUDA call, the theta
schemes, the binding's checks, and the struct layouts the binding shares with the header."""
from __future__ import annotations

import ctypes
import math
import shutil
import subprocess

import numpy as np
import pytest
import torch

from conftest import ROOT


@pytest.fixture()
def buf():
    return (ctypes.c_double * 64)()


def rope_args(ops, p, **changes):
    """A valid call on made-up addresses (never dereferenced: what is refused never launches)."""
    q = ops.RopeTensor(p, p + 128, 2, 32, 16, 8, 32, 16, 8)
    k = ops.RopeTensor(p, p + 256, 2, 32, 16, 8, 32, 16, 8)
    r = ops.Rope(q, k, 2, 2, 8, 8, p, None, 0, 0, 0, ops.DTYPE_F32, 0, 1.0)
    for name, value in changes.items():
        target, _, field = name.rpartition("__")
        setattr(getattr(r, target) if target else r, field, value)
    return r


ROPE_REFUSALS = [
    ({"dtype": 2}, "dtype"), ({"dtype": 4}, "dtype"), ({"batch": -1}, "negative size"),
    ({"tokens": 1 << 31}, "too large"), ({"rotary_dim": 3}, "rotary_dim"), ({"rotary_dim": 0}, "rotary_dim"),
    ({"rotary_dim": 10}, "rotary_dim"), ({"magnitude": math.inf}, "magnitude"), ({"theta": None}, "theta is null"),
    ({"q__in_": None}, "q: required pointer"), ({"k__out": None}, "k: required pointer"),
    ({"q__heads": -1}, "head count"), ({"q__in_stride_head": -8}, "negative stride"),
    ({"q__out_stride_head": 4}, "overlap"), ({"k__out_stride_batch": 0}, "overlap"),
    ({"q__in_stride_batch": 1 << 61}, "stride too large"), ({"flags": 4}, "unknown flag"),
    ({"position_stride_token": -1, "positions": 8}, "negative position stride"),
]


@pytest.mark.parametrize("changes,message", ROPE_REFUSALS)
def test_rope_refuses(ops, buf, changes, message):
    p = ctypes.addressof(buf)
    assert ops.lib().levo_rope_qk(ctypes.byref(rope_args(ops, p, **changes)), None) == ops.EINVAL
    assert message in ops.last_error()


def test_rope_refuses_misaligned_pointers_and_other_strides_in_place(ops, buf):
    p = ctypes.addressof(buf)
    lib = ops.lib()
    for changes in ({"theta": p + 4}, {"positions": p + 4}, {"q__in_": p + 2}, {"k__out": p + 1}):
        assert lib.levo_rope_qk(ctypes.byref(rope_args(ops, p, **changes)), None) == ops.EINVAL
        assert "aligned" in ops.last_error()
    r = rope_args(ops, p, q__out=p, q__out_stride_batch=64)
    assert lib.levo_rope_qk(ctypes.byref(r), None) == ops.EINVAL
    assert "in place" in ops.last_error()
    assert lib.levo_rope_qk(None, None) == ops.EINVAL
    r = rope_args(ops, p, batch=(1 << 31) - 1, tokens=(1 << 31) - 1, q__heads=0, k__in_stride_batch=0,
                  k__out_stride_batch=0)
    assert lib.levo_rope_qk(ctypes.byref(r), None) == ops.EINVAL  # a broadcast output


def test_rope_limits(ops, buf):
    p = ctypes.addressof(buf)
    lib = ops.lib()
    wide = dict(head_dim=8194, rotary_dim=8, q__heads=1, k__heads=0, batch=1, tokens=1)
    assert lib.levo_rope_qk(ctypes.byref(rope_args(ops, p, **wide)), None) == ops.EUNSUPPORTED
    assert "8192" in ops.last_error()
    far = dict(batch=1 << 16, tokens=1 << 16, k__heads=0, q__heads=1, q__in_stride_batch=0, q__in_stride_token=0,
               q__out_stride_batch=1 << 20, q__out_stride_token=16)
    assert lib.levo_rope_qk(ctypes.byref(rope_args(ops, p, **far)), None) == ops.EUNSUPPORTED
    assert "too many tokens" in ops.last_error()


def test_rope_refuses_outputs_that_are_another_tensors(ops, buf):
    p = ctypes.addressof(buf)
    lib = ops.lib()
    for changes in ({"k__out": p + 128}, {"q__in_": p + 256}, {"k__in_": p + 128}):
        assert lib.levo_rope_qk(ctypes.byref(rope_args(ops, p, **changes)), None) == ops.EINVAL
        assert "another tensor's" in ops.last_error()
    for out, start in ((p + 256, p), (p + 128, p), (p + 384, p + 256)):  # k's cache, q's output, v in k's cache
        v = ops.RopeTensor(start, out, 2, 32, 16, 8, 32, 16, 8)
        a = ops.RopeAppend(rope_args(ops, p), v, 8, 2, p, None, None)
        assert lib.levo_rope_append_kv(ctypes.byref(a), None) == ops.EINVAL
        assert "another tensor's" in ops.last_error()


def apart_args(ops, p):
    """A valid call whose tensors lie apart: 256 bytes each, from 4096 bytes on."""
    q = ops.RopeTensor(p + 4096, p + 8192, 2, 32, 16, 8, 32, 16, 8)
    k = ops.RopeTensor(p + 12288, p + 16384, 2, 32, 16, 8, 32, 16, 8)
    return rope_args(ops, p, q=q, k=k)


@pytest.mark.parametrize("changes,message", [
    ({"q__out": 4096 + 4}, "its own input"),            # one element on
    ({"q__out": 4096 - 64}, "its own input"),           # out = buf[:, :-1], in = buf[:, 1:]
    ({"q__out": 4096 + 252}, "its own input"),          # the last element alone
    ({"q__out": 4096 - 252}, "its own input"),
    ({"q__out": 4096 + 32, "q__in_stride_head": 16, "q__in_stride_token": 32, "q__in_stride_batch": 64,
      "q__out_stride_head": 32, "q__out_stride_token": 8, "q__out_stride_batch": 64}, "its own input"),
    ({"q__out": 4096 + 28, "q__in_stride_batch": 0, "q__in_stride_token": 0, "q__in_stride_head": 0}, "its own input"),
    ({"k__out": 8192 + 252}, "another tensor's"), ({"k__out": 4096 - 252}, "another tensor's"),
    ({"q__out": 12288 + 128}, "another tensor's"),
    ({"k__in_": 8192 + 32, "k__in_stride_head": 0}, "another tensor's"),
])
def test_rope_refuses_outputs_that_overlap(ops, buf, changes, message):
    p = ctypes.addressof(buf)
    r = apart_args(ops, p)
    for name, value in changes.items():
        target, _, field = name.rpartition("__")
        setattr(getattr(r, target), field, p + value if field in ("in_", "out") else value)
    assert ops.lib().levo_rope_qk(ctypes.byref(r), None) == ops.EINVAL
    assert message in ops.last_error(), ops.last_error()


def test_append_refuses_caches_that_overlap(ops, buf):
    p = ctypes.addressof(buf)
    for k_in, k_out, v_in, v_out, message in (
            (12288, 12288 - 64, 20480, 24576, "its own input"),     # tokens that lie in rows 1 and 2 of the cache
            (12288, 16384, 20480, 20480 - 64, "its own input"),
            (12288, 16384, 20480, 16384 + 508, "another tensor's"),  # the caches' ends
            (12288, 16384, 16384 + 64, 24576, "another tensor's"),   # v in a row of k's cache
            (12288, 8192 + 32, 20480, 24576, "another tensor's")):
        r = apart_args(ops, p)
        r.k = ops.RopeTensor(p + k_in, p + k_out, 2, 32, 16, 8, 64, 16, 8)
        v = ops.RopeTensor(p + v_in, p + v_out, 2, 32, 16, 8, 64, 16, 8)
        a = ops.RopeAppend(r, v, 8, 4, p, None, None)
        assert ops.lib().levo_rope_append_kv(ctypes.byref(a), None) == ops.EINVAL
        assert message in ops.last_error(), ops.last_error()


def test_which_layouts_overlap(tmp_path):
    """csrc/strided.h against sets of elements."""
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no host compiler")
    exe = tmp_path / "strided"
    subprocess.run([gxx, "-std=c++17", "-O2", "-I", str(ROOT / "levo2.cpp_b200" / "csrc"),
                    str(ROOT / "tests" / "cpp" / "strided_test.cpp"), "-o", str(exe)], check=True)
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0 and "strided: ok" in run.stdout, run.stdout


def test_rope_zero_sizes_are_noops(ops, buf):
    p = ctypes.addressof(buf)
    lib = ops.lib()
    for changes in ({"batch": 0}, {"tokens": 0}, {"q__heads": 0, "k__heads": 0}):
        assert lib.levo_rope_qk(ctypes.byref(rope_args(ops, p, **changes)), None) == ops.OK
    r = ops.RopeAppend(rope_args(ops, p, batch=0), ops.RopeTensor(), 0, 4, p, None, None)
    assert lib.levo_rope_append_kv(ctypes.byref(r), None) == ops.OK


def test_append_refuses(ops, buf):
    p = ctypes.addressof(buf)
    lib = ops.lib()

    def call(message, rope=None, v=None, v_dim=8, capacity=2, lengths=p, counts=None, status=None):
        v = ops.RopeTensor(p, p + 128, 2, 32, 16, 8, 32, 16, 8) if v is None else v
        a = ops.RopeAppend(rope_args(ops, p) if rope is None else rope, v, v_dim, capacity, lengths, counts, status)
        assert lib.levo_rope_append_kv(ctypes.byref(a), None) == ops.EINVAL
        assert message in ops.last_error(), ops.last_error()

    call("unknown flag", rope=rope_args(ops, p, flags=ops.ROPE_ADJOINT))
    call("capacity", capacity=-1)
    call("v_dim", v_dim=0)
    call("overlap", capacity=3)  # three rows of 16 do not fit a batch stride of 32
    call("lengths is null", lengths=None)
    call("aligned", lengths=p + 4)
    call("aligned", counts=p + 4)
    call("aligned", status=p + 2)
    call("its own input", v=ops.RopeTensor(p, p, 2, 32, 16, 8, 32, 16, 8))
    call("its own input", rope=rope_args(ops, p, k__out=p))
    assert lib.levo_rope_append_kv(None, None) == ops.EINVAL


def test_theta_schemes(ops):
    """Against the formulas in Python floats (pow and one or two further roundings: a few 2^-53)."""
    def close(got, want):
        assert got.dtype == torch.float64
        assert np.allclose(got.numpy(), np.asarray(want), rtol=1e-14, atol=0)

    for rot in (2, 64, 110, 128):
        plain = [10000.0 ** (-2 * i / rot) for i in range(rot // 2)]
        close(ops.rope_theta(rot), plain)
        close(ops.rope_theta(rot, base=5e5), [5e5 ** (-2 * i / rot) for i in range(rot // 2)])
        close(ops.rope_theta(rot, scaling="linear", factor=8.0), [t / 8 for t in plain])
        if rot > 2:
            base = 10000.0 * 8.0 ** (rot / (rot - 2))
            close(ops.rope_theta(rot, scaling="ntk", factor=8.0), [base ** (-2 * i / rot) for i in range(rot // 2)])
        want = []
        for t in plain:
            g = min(max((4096 * t / (2 * math.pi) - 1) / (32 - 1), 0.0), 1.0)
            want.append((1 - g) * t / 8 + g * t)
        close(ops.rope_theta(rot, scaling="by_parts", factor=8.0, context=4096), want)


@pytest.mark.parametrize("kw,message", [
    ({"rotary_dim": 0}, "rotary_dim"), ({"rotary_dim": 7}, "rotary_dim"), ({"rotary_dim": -2}, "rotary_dim"),
    ({"rotary_dim": 8, "base": 0.0}, "base"), ({"rotary_dim": 8, "base": math.nan}, "base"),
    ({"rotary_dim": 8, "scaling": "linear", "factor": 0.5}, "factor"),
    ({"rotary_dim": 2, "scaling": "ntk", "factor": 2.0}, "NTK"),
    ({"rotary_dim": 8, "scaling": "by_parts", "factor": 2.0, "context": 0.0}, "context"),
    ({"rotary_dim": 8, "scaling": "by_parts", "factor": 2.0, "slow": 4.0, "fast": 4.0}, "slow < fast"),
    ({"rotary_dim": 8, "scaling": "other"}, "scaling must be one of"),
])
def test_theta_refuses(ops, kw, message):
    with pytest.raises(ValueError, match=message):
        ops.rope_theta(**kw)


@pytest.mark.parametrize("kw", [{"rotary_dim": 4, "factor": 1e200}, {"rotary_dim": 64, "base": 1e300, "factor": 1e9}])
def test_theta_refuses_a_base_that_overflows(ops, kw):
    """base * factor^(n / (n - 2)) beyond the range of 64 bits would give 0 for every pair but the first."""
    with pytest.raises(ValueError, match="scaled base"):
        ops.rope_theta(scaling="ntk", **kw)
    large = ops.rope_theta(4, base=1e4, scaling="ntk", factor=1e150)
    assert np.allclose(large.numpy(), [1.0, 1e-152], rtol=1e-14, atol=0)


def sampling_args(ops, p, **changes):
    s = ops.Sampling(p, 2, 16, 16, p, None, None, None, None, 0, None, 0, 0, None, 0, 0, p, None, None, 1.0, 1.0, 0.0,
                     1.0, ops.DTYPE_F32)
    for name, value in changes.items():
        setattr(s, name, value)
    return s


@pytest.mark.parametrize("changes,message", [
    ({"dtype": 2}, "dtype"), ({"rows": -1}, "negative size"), ({"vocab": 0}, "empty vocabulary"),
    ({"ld": 15}, "row stride"), ({"logits": None}, "null"), ({"uniforms": None}, "null"), ({"tokens_out": None}, "null"),
    ({"temperature": -1.0}, "temperature"), ({"temperature": math.nan}, "temperature"),
    ({"temperature": math.inf}, "temperature"), ({"top_k": -1}, "top_k"), ({"top_p": 1.5}, "top_p"),
    ({"top_p": math.nan}, "top_p"), ({"min_p": -0.1}, "min_p"), ({"streams": -1}, "negative size"),
    ({"recent": 8, "recent_len": 1, "penalty": 0.0}, "penalty"), ({"n_ignore": 1}, "ignore list is null"),
    ({"tokens_out": 4}, "aligned"), ({"logprob_out": 2}, "aligned"), ({"temperature_rows": 2}, "aligned"),
])
def test_sample_refuses(ops, buf, changes, message):
    s = sampling_args(ops, ctypes.addressof(buf), **changes)
    assert ops.lib().levo_sample_tokens(ctypes.byref(s), None) == ops.EINVAL
    assert message in ops.last_error()


def test_sample_limits(ops, buf):
    p = ctypes.addressof(buf)
    lib = ops.lib()
    assert lib.levo_sample_tokens(ctypes.byref(sampling_args(ops, p, rows=0)), None) == ops.OK
    assert lib.levo_sample_tokens(ctypes.byref(sampling_args(ops, p, vocab=131073, ld=131073)),
                                  None) == ops.EUNSUPPORTED
    assert lib.levo_sample_tokens(None, None) == ops.EINVAL


def test_binding_refuses_what_the_library_cannot_see(ops):
    q = torch.zeros((1, 2, 2, 8))
    theta = torch.zeros(4, dtype=torch.float64)
    with pytest.raises(ValueError, match="CUDA"):
        ops.rope_qk_t(q, q, theta)
    with pytest.raises(ValueError, match="float64"):
        ops.rope_qk_t(q, q, theta.float())
    with pytest.raises(ValueError, match="int64"):
        ops.rope_qk_t(q, q, theta, torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="positions must be"):
        ops.rope_qk_t(q, q, theta, torch.zeros(3, dtype=torch.int64))
    with pytest.raises(ValueError, match="share a dtype"):
        ops.rope_qk_t(q, q.half(), theta)
    with pytest.raises(ValueError, match="batch and tokens"):
        ops.rope_qk_t(q, torch.zeros((1, 3, 2, 8)), theta)
    with pytest.raises(ValueError, match="unit stride"):
        ops.rope_qk_t(torch.zeros((1, 2, 8, 2)).transpose(2, 3), None, theta)
    with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
        ops.rope_qk_t(q.double(), q.double(), theta)
    cache = torch.zeros((1, 4, 2, 8))
    lengths = torch.zeros(1, dtype=torch.int64)
    with pytest.raises(ValueError, match="CUDA"):
        ops.rope_append_kv_t(q, q, q, theta, cache, cache.clone(), lengths)
    with pytest.raises(ValueError, match="share a capacity"):
        ops.rope_append_kv_t(q, q, q, theta, cache, torch.zeros((1, 5, 2, 8)), lengths)
    with pytest.raises(ValueError, match="lengths"):
        ops.rope_append_kv_t(q, q, q, theta, cache, cache.clone(), lengths.int())
    with pytest.raises(ValueError, match="k cache"):
        ops.rope_append_kv_t(q, q, q, theta, torch.zeros((1, 4, 1, 8)), cache, lengths)
    x, u = torch.zeros((2, 5)), torch.zeros(2)
    with pytest.raises(ValueError, match="CUDA"):
        ops.sample_tokens_t(x, u)
    with pytest.raises(ValueError, match="uniforms"):
        ops.sample_tokens_t(x, torch.zeros(3))
    with pytest.raises(ValueError, match="per-row setting"):
        ops.sample_tokens_t(x, u, top_k=torch.zeros(2))
    with pytest.raises(ValueError, match="recent"):
        ops.sample_tokens_t(x, u, recent=torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="unit stride"):
        ops.sample_tokens_t(torch.zeros((5, 2)).t(), u)


def test_struct_layouts_match_the_header(ops, tmp_path):
    """sizeof and every field's offset, as a C compiler sees them."""
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("no host compiler")
    c_names = {"in_": "in"}
    for i, axis in enumerate(("batch", "token", "head")):
        c_names |= {f"in_stride_{axis}": f"in_stride[{i}]", f"out_stride_{axis}": f"out_stride[{i}]"}
    c_names |= {"position_stride_batch": "position_stride[0]", "position_stride_token": "position_stride[1]"}
    structs = {"levo_rope_tensor": ops.RopeTensor, "levo_rope": ops.Rope, "levo_rope_append": ops.RopeAppend,
               "levo_sampling": ops.Sampling}
    lines, want = [], []
    for name, cls in structs.items():
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        want.append(ctypes.sizeof(cls))
        for field, _ in cls._fields_:
            lines.append(f'printf("%zu\\n", offsetof({name}, {c_names.get(field, field)}));')
            want.append(getattr(cls, field).offset)
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include "levo_ops.h"\nint main(void) {\n' + "\n".join(lines) + "\nreturn 0; }\n")
    subprocess.run([gcc, "-std=gnu99", "-I", str(ROOT / "include"), str(src), "-o", str(tmp_path / "layout")], check=True)
    got = subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout.split()
    assert [int(v) for v in got] == want
