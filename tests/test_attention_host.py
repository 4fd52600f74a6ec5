"""Attention operators without a GPU: what they refuse, and the parameters that they hand to the library."""
import ctypes
import math
import re
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

import kermac_amd as kermac
from kermac_amd import _backend
from kermac_amd.attention import _plan_attention, _plan_attention_grad

ROOT = Path(__file__).resolve().parents[1]


def make(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


def plan(q, k, v, out=None, scale=None, key_lengths=None, key_mask=None, return_lse=False, prefix=None):
    return _plan_attention(q, k, v, out, scale, key_lengths, key_mask, return_lse, prefix=prefix, require_device=False)


def test_operands_on_the_cpu_are_refused():
    q = make(1, 2, 2, 8)
    with pytest.raises(ValueError, match="CUDA device"):
        kermac.cross_attention(q, q, q)
    with pytest.raises(ValueError, match="CUDA device"):
        kermac.prefix_attention(q, q[0], q[0], q, q, torch.zeros(1, dtype=torch.int32))


@pytest.mark.parametrize("error, match, change", [
    (TypeError, "PyTorch tensor", dict(q=3.0)),
    (TypeError, "PyTorch tensor", dict(k=[1.0])),
    (TypeError, "dtype", dict(q=make(2, 5, 4, 16, dtype=torch.float64))),
    (TypeError, "dtype", dict(k=make(2, 7, 2, 16, dtype=torch.bfloat16))),
    (TypeError, "dtype", dict(v=make(2, 7, 2, 24, dtype=torch.float16))),
    (ValueError, "3-dimensional or 4-dimensional", dict(q=make(5, 16))),
    (ValueError, "3-dimensional or 4-dimensional", dict(v=make(1, 2, 7, 2, 24))),
    (ValueError, "batch size", dict(k=make(3, 7, 2, 16), v=make(3, 7, 2, 24))),
    (ValueError, "batch size", dict(k=make(1, 7, 2, 16))),
    (ValueError, "batch size", dict(q=make(1, 5, 4, 16))),
    (ValueError, "features", dict(k=make(2, 7, 2, 17))),
    (ValueError, "tokens and heads", dict(v=make(2, 8, 2, 24))),
    (ValueError, "tokens and heads", dict(v=make(2, 7, 4, 24))),
    (ValueError, "multiple of the heads", dict(q=make(2, 5, 3, 16))),
    (ValueError, "multiple of the heads", dict(k=make(2, 7, 0, 16), v=make(2, 7, 0, 24))),
    (ValueError, "1 .. 256", dict(q=make(2, 5, 4, 257), k=make(2, 7, 2, 257))),
    (ValueError, "1 .. 256", dict(v=make(2, 7, 2, 0))),
    (ValueError, "stride 1", dict(q=make(2, 5, 16, 4).transpose(2, 3))),
    (ValueError, "finite", dict(scale=math.inf)),
    (ValueError, "finite", dict(scale=math.nan)),
    (TypeError, "torch.int32", dict(key_lengths=torch.zeros(2, dtype=torch.int64))),
    (ValueError, "key_lengths", dict(key_lengths=torch.zeros(1, dtype=torch.int32))),
    (ValueError, "key_lengths", dict(key_lengths=torch.zeros(4, dtype=torch.int32)[::2])),
    (TypeError, "torch.bool", dict(key_mask=torch.zeros(2, 7))),
    (ValueError, "key_mask", dict(key_mask=torch.zeros(2, 8, dtype=torch.bool))),
    (ValueError, "key_mask", dict(key_mask=torch.zeros(3, 7, dtype=torch.bool))),
    (TypeError, "dtype", dict(out=make(2, 5, 4, 24, dtype=torch.float16))),
    (ValueError, "shape", dict(out=make(2, 5, 4, 16))),
    (ValueError, "stride 1", dict(out=make(2, 5, 24, 4).transpose(2, 3))),
    (ValueError, "expanded", dict(out=make(1, 5, 4, 24).expand(2, 5, 4, 24))),
], ids=lambda x: None if isinstance(x, type) else str(x) if isinstance(x, str) else "-".join(x))
def test_refusals(error, match, change):
    arguments = dict(q=make(2, 5, 4, 16), k=make(2, 7, 2, 16), v=make(2, 7, 2, 24))
    plan(**arguments)
    arguments.update(change)
    with pytest.raises(error, match=match):
        plan(**arguments)


@pytest.mark.parametrize("error, match, change", [
    (ValueError, "no batch mode", dict(prefix=(make(1, 9, 2, 16), make(9, 2, 24)))),
    (ValueError, "prefix_keys", dict(prefix=(make(9, 1, 16), make(9, 2, 24)))),
    (ValueError, "prefix_keys", dict(prefix=(make(9, 2, 8), make(9, 2, 24)))),
    (ValueError, "prefix_values", dict(prefix=(make(9, 2, 16), make(8, 2, 24)))),
    (ValueError, "prefix_values", dict(prefix=(make(9, 2, 16), make(9, 2, 16)))),
    (TypeError, "dtype", dict(prefix=(make(9, 2, 16, dtype=torch.float16), make(9, 2, 24)))),
    (ValueError, "batch size", dict(k=make(1, 7, 2, 16), v=make(1, 7, 2, 24))),
    (ValueError, "lengths", dict(key_lengths=torch.zeros(3, dtype=torch.int32))),
], ids=lambda x: None if isinstance(x, type) else str(x) if isinstance(x, str) else "-".join(x))
def test_prefix_refusals(error, match, change):
    arguments = dict(q=make(2, 5, 4, 16), k=make(2, 7, 2, 16), v=make(2, 7, 2, 24), prefix=(make(9, 2, 16), make(9, 2, 24)),
                     key_lengths=torch.zeros(2, dtype=torch.int32))
    plan(**arguments)
    arguments.update(change)
    with pytest.raises(error, match=match):
        plan(**arguments)


def test_parameters_of_views():
    both = make(2, 7, 2, 3, 16)
    q = make(2, 4, 5, 16).transpose(1, 2)
    out = make(2, 5, 4, 20)[..., :16]
    params = plan(q, both[:, :, 0, :2], both[:, :, 1, :2], out=out, scale=0.5).params
    assert (params.type, params.l, params.m, params.n, params.h, params.g, params.k, params.o) == (_backend.FP32, 2, 5, 7, 4, 2, 16, 16)
    assert (params.q_ls, params.q_ms, params.q_hs) == (320, 16, 80)
    assert (params.key_ls, params.key_ns, params.key_gs) == (672, 96, 16)
    assert params.value == params.key + 48 * 4 and params.scale == 0.5
    assert (params.out_ls, params.out_ms, params.out_hs) == (400, 80, 20)
    params = plan(q, both[:1, :, 0, :2], both[:1, :, 1, :2], key_mask=torch.ones(7, dtype=torch.bool)).params
    assert params.key_ls == params.value_ls == params.key_mask_ls == 0 and params.key_mask_ns == 1
    assert params.scale == 0.25


def library_parameters(**change):
    params = plan(make(2, 5, 4, 16), make(2, 7, 2, 16), make(2, 7, 2, 24), key_lengths=torch.zeros(2, dtype=torch.int32),
                  prefix=(make(9, 2, 16), make(9, 2, 24))).params
    for name, value in change.items():
        setattr(params, name, value)
    return params


@pytest.mark.parametrize("change", [
    dict(type=3), dict(l=-1), dict(n=-1), dict(n=2**31 - 1), dict(h=5), dict(g=0), dict(k=0), dict(k=257), dict(o=257), dict(scale=math.nan),
    dict(q_ms=-1), dict(prefix_value_gs=-1), dict(prefix_n=-1), dict(q=None), dict(out=None), dict(key=None), dict(prefix_value=None),
    dict(key_lengths=None), dict(key_mask=1), dict(l=2**20, m=2**20),
], ids=lambda c: "-".join(f"{k}={v}" for k, v in c.items()))
def test_the_library_refuses_before_any_device_call(change):
    assert _backend.attention_workspace_bytes(library_parameters()) > 0
    params = library_parameters(**change)
    for call in (lambda: _backend.attention(params, None), lambda: _backend.attention_workspace_bytes(params)):
        with pytest.raises(_backend.BackendError) as info:
            call()
        assert info.value.status == _backend.ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("error, match, change", [
    (TypeError, "grad_out", dict(grad_out=None)),
    (TypeError, "grad_out", dict(grad_out=make(2, 5, 4, 24, dtype=torch.float16))),
    (ValueError, "grad_out", dict(grad_out=make(2, 5, 4, 16))),
    (ValueError, "grad_out", dict(grad_out=make(2, 5, 24, 4).transpose(2, 3))),
    (ValueError, "out", dict(out=make(2, 5, 4, 16))),
    (TypeError, "lse", dict(lse=make(2, 5, 4, dtype=torch.float64))),
    (ValueError, "lse", dict(lse=make(2, 4, 5))),
    (ValueError, "lse", dict(lse=make(2, 4, 5).transpose(1, 2))),
    (ValueError, "batch size", dict(keys=make(1, 7, 2, 16))),
    (TypeError, "torch.int32", dict(key_lengths=torch.zeros(2))),
], ids=lambda x: None if isinstance(x, type) else str(x) if isinstance(x, str) else "-".join(x))
def test_gradient_refusals(error, match, change):
    arguments = dict(grad_out=make(2, 5, 4, 24), queries=make(2, 5, 4, 16), keys=make(2, 7, 2, 16), values=make(2, 7, 2, 24), out=make(2, 5, 4, 24),
                     lse=make(2, 5, 4), scale=None, key_lengths=None, key_mask=None, require_device=False)
    plan = _plan_attention_grad(**arguments)
    assert [tuple(x.shape) for x in plan.out] == [(2, 5, 4, 16), (2, 7, 2, 16), (2, 7, 2, 24)]
    arguments.update(change)
    with pytest.raises(error, match=match):
        _plan_attention_grad(**arguments)


@pytest.mark.parametrize("change", [
    dict(type=-1), dict(m=-1), dict(h=3), dict(k=0), dict(o=257), dict(scale=math.inf), dict(key_entries=3), dict(key_entries=1), dict(grad_out_ls=-1),
    dict(lse=None), dict(grad_q=None), dict(grad_value=None), dict(value=None), dict(out=None),
], ids=lambda c: "-".join(f"{k}={v}" for k, v in c.items()))
def test_the_library_refuses_gradients_before_any_device_call(change):
    params = _plan_attention_grad(make(2, 5, 4, 24), make(2, 5, 4, 16), make(2, 7, 2, 16), make(2, 7, 2, 24), make(2, 5, 4, 24), make(2, 5, 4), None, None, None,
                                  require_device=False).params
    needed = _backend.attention_gradient_workspace_bytes(params)
    assert needed >= 8 * (2 * 5 * 4 + 1)
    for workspace, nbytes in ((None, needed), (1 << 20, 8 * (2 * 5 * 4 + 1) - 1), ((1 << 20) + 4, needed)):
        params.workspace, params.workspace_bytes = workspace, nbytes
        with pytest.raises(_backend.BackendError, match="workspace"):
            _backend.attention_gradient(params, None)
    for name, value in change.items():
        setattr(params, name, value)
    with pytest.raises(_backend.BackendError) as info:
        _backend.attention_gradient_workspace_bytes(params)
    assert info.value.status == _backend.ERR_INVALID_ARGUMENT


def test_header_and_binding_agree(tmp_path):
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("no C compiler")
    structs = {"kmc_attention_params": _backend.AttentionParams, "kmc_attention_gradient_params": _backend.AttentionGradientParams}
    lines = ['#include "kermac_amd.h"', "#include <stddef.h>", "#include <stdio.h>", "int main(void) {"]
    for c_name, binding in structs.items():
        lines.append(f'  printf("{c_name} size %zu\\n", sizeof({c_name}));')
        lines += [f'  printf("{c_name} {field} %zu\\n", offsetof({c_name}, {field}));' for field, _ in binding._fields_]
    lines += ['  printf("types %d %d %d\\n", KMC_FP32, KMC_FP16, KMC_BF16);', "  return 0;", "}"]
    (tmp_path / "probe.c").write_text("\n".join(lines))
    subprocess.run([gcc, "-std=c11", "-Wall", "-Werror", f"-I{ROOT / 'include'}", str(tmp_path / "probe.c"), "-o", str(tmp_path / "probe")], check=True)
    printed = subprocess.run([str(tmp_path / "probe")], check=True, capture_output=True, text=True).stdout
    for c_name, binding in structs.items():
        assert f"{c_name} size {ctypes.sizeof(binding)}\n" in printed
        for field, _ in binding._fields_:
            assert re.search(rf"^{c_name} {field} {getattr(binding, field).offset}$", printed, re.M), f"{c_name}.{field}"
    assert f"types {_backend.FP32} {_backend.FP16} {_backend.BF16}\n" in printed


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("L, M, N, H, G, K, P, lengths", [(1, 1, 5000, 8, 8, 64, None, False), (3, 1, 4000, 16, 4, 128, None, True), (2, 300, 700, 4, 2, 80, None, False),
                                                          (64, 1, 500, 8, 2, 128, 8192, True), (2, 50, 60, 8, 1, 256, 1000, True)])
def test_the_workspace_that_is_asked_for_is_what_the_call_uses(dtype, L, M, N, H, G, K, P, lengths):
    """The sizes are asked for once per shape, by a call of that shape with other addresses: they have to be those of the call itself."""
    import importlib
    attention = importlib.import_module("kermac_amd.attention")
    q, k, v = make(L, M, H, K, dtype=dtype), make(L, N, G, K, dtype=dtype), make(L, N, G, K, dtype=dtype)
    prefix = (make(P, G, K, dtype=dtype), make(P, G, K, dtype=dtype)) if P else None
    of = plan(q, k, v, key_lengths=torch.zeros(L, dtype=torch.int32) if lengths else None, prefix=prefix)
    assert attention._workspace_bytes(*of.extents) == _backend.attention_workspace_bytes(of.params)
    if prefix is None:
        of = _plan_attention_grad(q, q, k, v, q, make(L, M, H), None, None, None, require_device=False)
        assert attention._gradient_workspace_bytes(*of.extents) == _backend.attention_gradient_workspace_bytes(of.params)


@pytest.mark.parametrize("scale", [1e39, -1e39, 3e38, -math.inf])
def test_scales_that_fp32_does_not_hold_to_base_2(scale):
    """Scores are taken to base 2: a scale is refused where fp32 does not hold its product with log2(e), in Python and in the library."""
    q, k, v = make(2, 5, 4, 16), make(2, 7, 2, 16), make(2, 7, 2, 24)
    with pytest.raises(ValueError, match="scale"):
        plan(q, k, v, scale=scale)
    with pytest.raises(ValueError, match="scale"):
        _plan_attention_grad(make(2, 5, 4, 24), q, k, v, make(2, 5, 4, 24), make(2, 5, 4), scale, None, None, require_device=False)
    assert plan(q, k, v, scale=-1.9e38).params.scale < -1.8e38
    assert _backend.attention_workspace_bytes(library_parameters(scale=-1.9e38)) > 0
    params = library_parameters(scale=scale)
    with pytest.raises(_backend.BackendError, match="scale"):
        _backend.attention(params, None)


def test_a_batch_of_no_sequences():
    """Empty tensors have no address, the lengths of a batch of none among them: the library takes that for a call with nothing to do."""
    params = plan(make(0, 5, 4, 16), make(0, 7, 2, 16), make(0, 7, 2, 24), key_lengths=torch.zeros(0, dtype=torch.int32), prefix=(make(9, 2, 16), make(9, 2, 24))).params
    assert params.key_lengths is None and params.causal == 1
    assert _backend.attention_workspace_bytes(params) == 0
    _backend.attention(params, None)


def test_operands_on_another_device_are_refused():
    q, k, v = make(2, 5, 4, 16), make(2, 7, 2, 16), make(2, 7, 2, 24)
    elsewhere = torch.device("meta")
    for change in (dict(k=k.to(elsewhere)), dict(v=v.to(elsewhere)), dict(out=make(2, 5, 4, 24).to(elsewhere)),
                   dict(key_lengths=torch.zeros(2, dtype=torch.int32, device=elsewhere)), dict(key_mask=torch.zeros(7, dtype=torch.bool, device=elsewhere)),
                   dict(prefix=(make(9, 2, 16).to(elsewhere), make(9, 2, 24)), key_lengths=torch.zeros(2, dtype=torch.int32))):
        with pytest.raises(ValueError, match="same CUDA device"):
            plan(**{**dict(q=q, k=k, v=v), **change})
    with pytest.raises(ValueError, match="same CUDA device"):
        _plan_attention_grad(make(2, 5, 4, 24), q, k, v, make(2, 5, 4, 24), make(2, 5, 4).to(elsewhere), None, None, None, require_device=False)


def test_the_workspace_of_a_gradient_has_room_for_shifts():
    """12 bytes per row and 4 per 128 rows of a head of keys: row statistics, and what is subtracted from the scores of rows whose lse is large."""
    plan = _plan_attention_grad(make(3, 50, 8, 24), make(3, 50, 8, 16), make(3, 7, 2, 16), make(3, 7, 2, 24), make(3, 50, 8, 24), make(3, 50, 8), None, None, None,
                                require_device=False)
    rows = 3 * 50 * 8
    assert _backend.attention_gradient_workspace_bytes(plan.params) >= 8 * rows + 16 + (4 * rows + 4 * 3 * 2 * 2 + 15) // 16 * 16


def test_a_prefix_alone_makes_the_own_keys_causal():
    """prefix_n > 0 with causal = 0 is the header's "prefix_n > 0 or causal": lengths are needed and a mask is refused, as with causal = 1."""
    assert _backend.attention_workspace_bytes(library_parameters(causal=0)) == _backend.attention_workspace_bytes(library_parameters()) > 0
    for change in (dict(key_lengths=None), dict(key_mask=16)):
        with pytest.raises(_backend.BackendError, match="prefix"):
            _backend.attention_workspace_bytes(library_parameters(causal=0, **change))


@pytest.mark.parametrize("L, M, N, H, G", [(8, 1, 32000, 32, 8), (16, 1, 8192, 32, 8), (1, 1, 32000, 8, 8), (128, 1, 8192, 32, 8), (2, 200, 3000, 8, 8)])
def test_lengths_do_not_change_the_parts(L, M, N, H, G):
    """How full the keys are is not known when the work is cut: a call with lengths is cut as one without."""
    q, k = make(1, M, H, 128, dtype=torch.bfloat16).expand(L, M, H, 128), make(1, N, G, 128, dtype=torch.bfloat16).expand(L, N, G, 128)
    out = torch.empty(L, M, H, 128, dtype=torch.bfloat16)
    with_lengths, without = (_backend.attention_workspace_bytes(plan(q, k, k, out=out, key_lengths=lengths).params) for lengths in (torch.zeros(L, dtype=torch.int32), None))
    assert with_lengths == without
