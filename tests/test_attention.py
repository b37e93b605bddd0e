"""cross_attention, its gradient and prefix_attention without a GPU: the oracle against autograd, the C-ABI's layout, what calls
are refused, and the plans."""
import ctypes
import glob
import math
import os
import re
import subprocess

import pytest
import torch

import kermac_b200 as kermac
from kermac_b200 import _native, attention
from oracle import attention_oracle as ao
from test_abi import ROOT

HEADER = os.path.join(ROOT, "include", "kermac_b200_attention.h")


def test_oracle_gradient_is_the_gradient_of_the_oracle():
    torch.manual_seed(0)
    L, N, M, H, Hk, D, scale = 2, 5, 7, 4, 2, 3, 0.7
    q, k, v = (torch.randn(L, n, h, D, dtype=torch.float64, requires_grad=True) for n, h in ((N, H), (M, Hk), (M, Hk)))
    lengths = [7, 4]
    s = torch.einsum("lnhd,lmhd->lhnm", q, k.repeat_interleave(2, dim=2)) * scale
    for l, n in enumerate(lengths):
        mask = torch.arange(M) >= n
        s = s.masked_fill(mask[None, None, None, :] & (torch.arange(L) == l)[:, None, None, None], -math.inf)
    out = torch.einsum("lhnm,lmhd->lnhd", torch.softmax(s, dim=-1), v.repeat_interleave(2, dim=2))
    g = torch.randn_like(out)
    grads = torch.autograd.grad(out, (q, k, v), g)
    f = [t.detach().float() for t in (q, k, v, g)]
    want, _, bound, _ = ao.attention(*f[:3], lengths, scale)
    assert (want - out.detach()).abs().max() < 1e-5
    found = ao.attention_grad(*f, lengths, scale)
    for name, grad in zip(("grad_q", "grad_k", "grad_v"), grads):
        assert (found[name][0] - grad).abs().max() < 1e-5
        assert found[name][1].shape == grad.shape and torch.all(found[name][1] < 1e-3)


def _c_args(**kw):
    """Arguments of a call that would be accepted; the pointers are never followed, because these tests launch nothing."""
    a = _native.KmAttentionArgs()
    a.l, a.n, a.m, a.heads, a.key_heads, a.d, a.type = 2, 3, 5, 4, 2, 8, _native.TYPE_BFLOAT16
    a.scale, a.q_batch, a.kv_batch = 0.5, 2, 2
    for name, rows, heads in (("q", 3, 4), ("k", 5, 2), ("v", 5, 2), ("out", 3, 4), ("grad_out", 3, 4), ("grad_q", 3, 4),
                              ("grad_k", 5, 2), ("grad_v", 5, 2), ("k_prefix", 6, 2), ("v_prefix", 6, 2)):
        setattr(a, name, _native.KmHeads(4096, rows * heads * 8, heads * 8, 8))
    a.lse, a.lse_stride_l, a.lse_stride_head = 4096, 12, 3
    for name, value in kw.items():
        if isinstance(value, tuple):
            tensor = getattr(a, name)
            setattr(tensor, *value)
            setattr(a, name, tensor)
        else:
            setattr(a, name, value)
    return a


REFUSED = [
    (dict(l=-1), 0, -2), (dict(n=-1), 1, -2), (dict(m=-1), 2, -2), (dict(prefix=-1), 1, -2), (dict(prefix=3), 0, -2),
    (dict(prefix=3), 2, -2), (dict(key_heads=0), 0, -2), (dict(key_heads=3), 0, -2), (dict(d=0), 0, -2), (dict(d=257), 2, -2),
    (dict(type=3), 0, -4), (dict(type=-1), 0, -4), (dict(scale=math.nan), 0, -5), (dict(scale=math.inf), 0, -5),
    (dict(scale=-1.0), 2, -5), (dict(q=("ptr", None)), 0, -1), (dict(k=("ptr", None)), 1, -1), (dict(v=("ptr", None)), 2, -1),
    (dict(out=("ptr", None)), 0, -1), (dict(lse=None), 2, -1), (dict(grad_out=("ptr", None)), 2, -1),
    (dict(grad_k=("ptr", None)), 2, -1), (dict(prefix=6, k_prefix=("ptr", None)), 1, -1),
    (dict(q=("stride_row", -8)), 0, -3), (dict(v=("stride_l", -8)), 2, -3), (dict(k=("stride_head", 1 << 40)), 0, -3),
    (dict(out=("stride_row", 8)), 0, -3), (dict(out=("stride_l", 0)), 0, -3), (dict(grad_v=("stride_head", 4)), 2, -3),
    (dict(lse_stride_head=2), 0, -3), (dict(lse_stride_l=-1), 1, -3), (dict(k=("stride_l", 0)), 0, -3),
    (dict(lengths=4096, lengths_stride=-1), 0, -3), (dict(q_batch=3), 2, -2), (dict(kv_batch=0), 2, -2),
    (dict(q_batch=1), 2, -3), (dict(kv_batch=1), 2, -3), (dict(m=(1 << 30) + 1), 0, -6), (dict(l=1 << 20, n=1 << 20), 0, -6),
]


@pytest.mark.parametrize("changes, kind, code", REFUSED, ids=str)
def test_the_c_abi_refuses(changes, kind, code):
    args = _c_args(**changes)
    assert getattr(_native.lib(), _native.ATTENTION_SYMBOLS[kind])(ctypes.byref(args), None) == code
    assert _native.last_error()
    assert _native.attention_scratch_bytes(args, kind) == 0
    with pytest.raises(ValueError):
        _native.launch_attention(args, kind, 0)
    with pytest.raises(ValueError):
        _native.describe_attention(args, kind)


PLANS = [           # what kernel takes a call: changes of _c_args, kind, a part of the description
    (dict(), 0, "own=few rows=8"),                                                 # 3 queries of 2 heads to a key head
    (dict(n=4), 0, "own=few rows=8"),
    (dict(n=8), 0, "own=few rows=16"),
    (dict(n=4, m=1100), 0, "own=few rows=8 tiles=1 splits=8 prefix=few rows=16 tiles=0 splits=0 scratch=0"),    # joined in a cluster
    (dict(n=9), 0, "own=tensor rows=256"),
    (dict(d=7, n=9), 0, "own=rows rows=64"),                                       # rows that TMA cannot copy
    (dict(d=7), 0, "own=scalar few"),
    (dict(d=136, n=9), 0, "own=rows"),
    (dict(k=("stride_row", 12)), 0, "own=scalar few"),
    (dict(v=("ptr", 4098)), 0, "own=scalar few"),
    (dict(type=0), 0, "own=scalar few"),
    (dict(type=0, n=9), 0, "own=rows"),                                            # 5 keys
    (dict(type=0, n=9, m=100), 0, "own=tensor32"),
    (dict(type=0, n=9, m=100, d=65), 0, "own=rows"),
    (dict(prefix=6), 1, "own=few rows=16 tiles=1 splits=1 prefix=few rows=16"),
    (dict(l=8, prefix=6), 1, "own=few rows=8 tiles=1 splits=1 prefix=few rows=8 tiles=6 splits=1"),        # 48 rows of a short prefix
    (dict(l=8, prefix=1 << 20), 1, "own=few rows=8 tiles=1 splits=1 prefix=tensor rows=256 tiles=1"),
    (dict(n=9, prefix=6), 1, "own=tensor rows=256 tiles=1 splits=1 prefix=tensor rows=256 tiles=1 splits=1"),
    (dict(), 2, "grad=tensor q_slices=1 kv_slices=1"),
    (dict(type=0), 2, "grad=rows"),
    (dict(d=7), 2, "grad=rows"),
    (dict(type=0, m=5000), 2, "q_slices=37"),                                      # 8 query tiles for 296 blocks
]


@pytest.mark.parametrize("changes, kind, expected", PLANS, ids=str)
def test_which_kernel_takes_a_call(changes, kind, expected):
    args = _c_args(**changes)
    if "n" in changes or "d" in changes or "m" in changes:                        # dense tensors of the new extents
        for name, rows, heads in (("q", args.n, 4), ("k", args.m, 2), ("v", args.m, 2), ("out", args.n, 4), ("grad_out", args.n, 4),
                                  ("grad_q", args.n, 4), ("grad_k", args.m, 2), ("grad_v", args.m, 2), ("k_prefix", 6, 2), ("v_prefix", 6, 2)):
            setattr(args, name, _native.KmHeads(4096, rows * heads * args.d, heads * args.d, args.d))
        args.lse_stride_l, args.lse_stride_head = 4 * args.n, args.n
    assert expected in _native.describe_attention(args, kind), _native.describe_attention(args, kind)


@pytest.mark.parametrize("kind", [0, 1, 2])
@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("changes", [dict(m=0), dict(n=0), dict(heads=0), dict(l=0, q_batch=0, kv_batch=0), dict(m=0, n=0)], ids=str)
def test_empty_extents_have_a_plan(kind, dtype, changes):
    args = _c_args(type=dtype, **changes)
    assert _native.describe_attention(args, kind)
    assert _native.attention_scratch_bytes(args, kind) >= 0


def test_scratch_is_bounded():
    # 2^27 rows of partial sums would be 34 GB: a single piece takes none
    args = _c_args(l=1, n=1 << 20, m=1 << 20, heads=1, key_heads=1, d=64)
    for name in ("q", "k", "v", "out"):
        setattr(args, name, _native.KmHeads(4096, 1 << 26, 64, 64))
    args.lse_stride_l, args.lse_stride_head = 1 << 20, 1 << 20
    assert _native.attention_scratch_bytes(args, 0) == 0
    args.type = _native.TYPE_FLOAT32                                              # 1.2 GB of planes: not asked for
    assert _native.attention_scratch_bytes(args, 0) == 0
    args.m = 1 << 10
    args.n = 1 << 10
    planes = 3 * (1 << 10) * 64 * 6
    pieces = args.m // 192                                                        # no piece is shorter than that: maximum, sum and 64 channels each
    assert planes <= _native.attention_scratch_bytes(args, 0) <= planes + pieces * (1 << 10) * 66 * 4 + 32


def test_the_c_abi_refuses_no_arguments_at_all():
    for kind in range(3):
        assert getattr(_native.lib(), _native.ATTENTION_SYMBOLS[kind])(None, None) == -1
        assert getattr(_native.lib(), _native.ATTENTION_SYMBOLS[3 + kind])(None) == 0
    assert _native.lib().kermac_b200_describe_attention(ctypes.byref(_c_args()), 3, None, 0) == -4
    assert _native.lib().kermac_b200_describe_attention(ctypes.byref(_c_args()), 0, None, 0) == -1


def test_calls_without_work_need_no_device():
    for kind, changes in ((0, dict(l=0)), (0, dict(n=0)), (1, dict(heads=0)), (2, dict(l=0, q_batch=0, kv_batch=0))):
        assert getattr(_native.lib(), _native.ATTENTION_SYMBOLS[kind])(ctypes.byref(_c_args(**changes)), None) == 0


def test_binding_matches_the_compiled_header(tmp_path):
    text = open(HEADER).read()
    body = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    assert set(re.findall(r"\b(kermac_b200_[a-z0-9_]+)\s*\(", body)) == set(_native.ATTENTION_SYMBOLS)
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "kermac_b200_attention.h"', 'int main(void) {']
    classes = {"KmHeads": _native.KmHeads, "KmAttentionArgs": _native.KmAttentionArgs}
    for name, cls in classes.items():
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        lines += [f'printf("{name} {f} %zu %zu\\n", offsetof({name}, {f}), sizeof((({name}*)0)->{f}));' for f, _ in cls._fields_]
    (tmp_path / "layout.c").write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(tmp_path / "layout.c"), "-o",
                    str(tmp_path / "layout")], check=True)
    got = [line.split() for line in subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.splitlines()]
    want = []
    for name, cls in classes.items():
        want.append([name, str(ctypes.sizeof(cls))])
        want += [[name, f, str(getattr(cls, f).offset), str(getattr(cls, f).size)] for f, _ in cls._fields_]
    assert got == want
    fields = re.findall(r"typedef struct KmAttentionArgs \{(.*?)\}", body, flags=re.S)[0]
    declared = [n.replace("*", "").split()[-1] for part in fields.split(";") if part.strip() for n in part.split(",")]
    assert declared == [f for f, _ in _native.KmAttentionArgs._fields_]


def _t(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


def _called(monkeypatch):
    monkeypatch.setattr(attention, "_is_cuda", lambda t: True)

    def launched(*args):
        raise AssertionError("the call was not refused")
    monkeypatch.setattr(attention, "_launch", launched)


def test_tensors_must_be_on_a_cuda_device():
    with pytest.raises(ValueError, match="CUDA device"):
        kermac.cross_attention(_t(2, 1, 8), _t(3, 1, 8), _t(3, 1, 8))
    with pytest.raises(TypeError, match="q must be a PyTorch tensor"):
        kermac.prefix_attention([1.0], _t(3, 1, 8), _t(3, 1, 8), _t(3, 1, 8), _t(3, 1, 8))


Q, K = (2, 3, 4, 8), (2, 5, 2, 8)
BAD_CROSS = [
    (dict(q=_t(3, 8)), ValueError, "dimensions"),
    (dict(q=_t(*Q, dtype=torch.float64)), TypeError, "dtype"),
    (dict(k=_t(*K, dtype=torch.bfloat16)), TypeError, "dtype"),
    (dict(v=None), TypeError, "v must be"),
    (dict(q=_t(2, 3, 8, 4).transpose(2, 3)), ValueError, "stride 1"),
    (dict(k=_t(2, 5, 2, 9)), ValueError, "channels"),
    (dict(q=_t(2, 3, 4, 300), k=_t(2, 5, 2, 300), v=_t(2, 5, 2, 300)), ValueError, r"\[1, 256\]"),
    (dict(v=_t(2, 6, 2, 8)), ValueError, "shape of k"),
    (dict(k=_t(2, 5, 3, 8), v=_t(2, 5, 3, 8)), ValueError, "multiple"),
    (dict(k=_t(2, 5, 0, 8), v=_t(2, 5, 0, 8)), ValueError, "multiple"),
    (dict(k=_t(3, 5, 2, 8), v=_t(3, 5, 2, 8)), ValueError, "batch size"),
    (dict(v=_t(1, 5, 2, 8).expand(2, 5, 2, 8)), ValueError, "both be broadcast"),
    (dict(lengths=[5, 5]), TypeError, "lengths"),
    (dict(lengths=_t(2)), TypeError, "int32"),
    (dict(lengths=_t(3, dtype=torch.int32)), ValueError, "lengths must have shape"),
    (dict(lengths=_t(2, 1, dtype=torch.int32)), ValueError, "lengths must have shape"),
    (dict(scale=-1.0), ValueError, "scale"),
    (dict(scale=math.nan), ValueError, "scale"),
    (dict(out=_t(2, 3, 4, 9)), ValueError, "out must have shape"),
    (dict(out=_t(3, 4, 8)), ValueError, "dimensions"),
    (dict(out=_t(*Q, dtype=torch.float16)), TypeError, "dtype"),
    (dict(lse=_t(2, 3, 4)), ValueError, "lse must have shape"),
    (dict(lse=_t(2, 4, 3, dtype=torch.float16)), TypeError, "lse must have dtype"),
    (dict(lse=_t(2, 3, 4).transpose(1, 2)), ValueError, "stride 1"),
]


@pytest.mark.parametrize("changes, error, match", BAD_CROSS, ids=lambda x: None if not isinstance(x, dict) else "-".join(x))
def test_cross_attention_refuses(changes, error, match, monkeypatch):
    _called(monkeypatch)
    given = dict(dict(q=_t(*Q), k=_t(*K), v=_t(*K)), **changes)
    with pytest.raises(error, match=match):
        kermac.cross_attention(given.pop("q"), given.pop("k"), given.pop("v"), **given)


BAD_PREFIX = [
    (dict(k_prefix=_t(1, 6, 2, 8)), ValueError, "dimensions"),
    (dict(k_prefix=_t(6, 2, 9)), ValueError, "k_prefix must have shape"),
    (dict(v_prefix=_t(6, 4, 8)), ValueError, "v_prefix must have shape"),
    (dict(v_prefix=_t(7, 2, 8)), ValueError, "shape of k_prefix"),
    (dict(v_prefix=_t(6, 2, 8, dtype=torch.float16)), TypeError, "dtype"),
]


@pytest.mark.parametrize("changes, error, match", BAD_PREFIX, ids=lambda x: None if not isinstance(x, dict) else "-".join(x))
def test_prefix_attention_refuses(changes, error, match, monkeypatch):
    _called(monkeypatch)
    given = dict(dict(q=_t(*Q), k_prefix=_t(6, 2, 8), v_prefix=_t(6, 2, 8), k=_t(*K), v=_t(*K)), **changes)
    with pytest.raises(error, match=match):
        kermac.prefix_attention(**given)


BAD_GRAD = [
    (dict(out=_t(3, 4, 8)), ValueError, "dimensions"),
    (dict(out=_t(2, 3, 4, 9)), ValueError, "out must have shape"),
    (dict(grad_out=_t(1, 3, 4, 8)), ValueError, "grad_out must have shape"),
    (dict(grad_out=_t(*Q, dtype=torch.bfloat16)), TypeError, "dtype"),
    (dict(lse=_t(2, 3, 4)), ValueError, "lse must have shape"),
    (dict(lse=None), TypeError, "lse"),
    (dict(grad_q=_t(1, 3, 4, 8)), ValueError, "grad_q must have shape"),
    (dict(grad_k=_t(5, 2, 8)), ValueError, "dimensions"),
    (dict(grad_v=_t(2, 2, 5, 8)), ValueError, "grad_v must have shape"),
    (dict(k=_t(1, 5, 2, 8)), ValueError, "shape of k"),
]


@pytest.mark.parametrize("changes, error, match", BAD_GRAD, ids=lambda x: None if not isinstance(x, dict) else "-".join(x))
def test_cross_attention_grad_refuses(changes, error, match, monkeypatch):
    _called(monkeypatch)
    given = dict(dict(q=_t(*Q), k=_t(*K), v=_t(*K), out=_t(*Q), lse=_t(2, 4, 3), grad_out=_t(*Q)), **changes)
    with pytest.raises(error, match=match):
        kermac.cross_attention_grad(**given)


def test_the_reference_name_serves_them():
    import kermac as served
    for name in ("cross_attention", "cross_attention_grad", "prefix_attention"):
        assert getattr(served, name) is getattr(kermac, name)


def test_the_extension_declines_what_is_not_an_ordinary_call():
    call = _native.torch_call()
    q, k = _t(*Q), _t(*K)
    assert call.attention(0, q, k, k, None, None, None, None, None, None, False) is None      # not on a CUDA device
    assert call.attention(2, q, k, k, None, None, None, None, None, None, False) is None
    assert call.attention(0, q.numpy(), k, k, None, None, None, None, None, None, False) is None
    assert call.attention(0, q, k) is None
    assert call.attention_grad(q, k, k, q, _t(2, 4, 3), q, None, None) is None
    assert call.attention_grad(None) is None


def _attention_kernels():
    """(name, parameters, body) of the kernels under csrc/attention."""
    for path in sorted(glob.glob(os.path.join(ROOT, "kermac_b200", "csrc", "attention", "*.cu*"))):
        text = re.sub(r"//[^\n]*|/\*.*?\*/", "", open(path).read(), flags=re.S)
        for head in re.finditer(r"__global__\s+void(?:\s+__launch_bounds__\((?:[^()]|\([^()]*\))*\))?\s+(\w+)\s*\(([^)]*)\)\s*\{", text):
            depth, end = 1, head.end()
            while depth:
                depth += {"{": 1, "}": -1}.get(text[end], 0)
                end += 1
            yield head.group(1), head.group(2), text[head.end():end]


def test_kernels_keep_the_order_of_overlapped_launches():
    kernels = list(_attention_kernels())
    assert len(kernels) >= 6
    for name, parameters, body in kernels:
        before, wait, _ = body.partition("after_previous_grid();")
        assert wait and "return;" not in before and "tmem_alloc" not in before, name
        assert "__restrict__" not in parameters + body and "__ldg" not in body, name


LONG = (1 << 32) + 1          # 1 in the 32 bits of the argument struct
TOO_LONG = [
    dict(q=_t(1, 4, 8).expand(LONG, 4, 8)),
    dict(q=_t(1, 3, 4, 8).expand(LONG, 3, 4, 8), k=_t(1, 5, 2, 8), v=_t(1, 5, 2, 8)),
    dict(q=_t(3, 1, 8).expand(3, LONG, 8), k=_t(5, 1, 8), v=_t(5, 1, 8)),
    dict(k=_t(2, 1, 2, 8).expand(2, LONG, 2, 8), v=_t(2, 1, 2, 8).expand(2, LONG, 2, 8)),
    dict(q=_t(3, 4, 8), k=_t(5, 2, 8), v=_t(5, 2, 8), lengths=_t(1, dtype=torch.int32).expand(LONG)),
    dict(k_prefix=_t(1, 2, 8).expand(LONG, 2, 8), v_prefix=_t(1, 2, 8).expand(LONG, 2, 8)),
]


@pytest.mark.parametrize("changes", TOO_LONG, ids="-".join)
def test_extents_beyond_the_argument_struct_are_refused(changes, monkeypatch):
    _called(monkeypatch)
    given = dict(dict(q=_t(*Q), k_prefix=_t(6, 2, 8), v_prefix=_t(6, 2, 8), k=_t(*K), v=_t(*K)), **changes)
    with pytest.raises(ValueError, match="below 2.31"):
        attention._marshal(given["q"], given["k"], given["v"], given.get("lengths"), None, prefix=(given["k_prefix"], given["v_prefix"]))


def test_a_scale_that_overflows_in_powers_of_two_is_refused():
    for kind in range(3):
        args = _c_args(scale=3.0e38)                                              # times log2(e): infinity
        assert getattr(_native.lib(), _native.ATTENTION_SYMBOLS[kind])(ctypes.byref(args), None) == -5
    assert _native.describe_attention(_c_args(scale=2.0e38), 0)


def test_pieces_are_planned_for_the_blocks_that_the_launch_has():
    # 4 tokens of 8 heads of 128, 1024 own keys below 4000 of a prefix: one launch of 32-key tiles, of which an SM holds one block, so that the
    # 32 blocks of own keys get 148 / 32 pieces, not the 296 / 32 of short keys alone
    args = _c_args(l=4, n=1, m=1024, heads=8, key_heads=8, d=128, prefix=4000)
    for name, rows in (("q", 1), ("out", 1), ("k", 1024), ("v", 1024), ("k_prefix", 4000), ("v_prefix", 4000)):
        setattr(args, name, _native.KmHeads(4096, rows * 8 * 128, 8 * 128, 128))
    args.lse_stride_l, args.lse_stride_head = 8, 1
    assert "own=few rows=8 tiles=1 splits=4 prefix=few rows=8 tiles=1 splits=18" in _native.describe_attention(args, 1)


def _big(**kw):
    """Dense tensors of the extents; nothing is launched."""
    args = _c_args(**kw)
    l, d, Hk = args.l, args.d, args.key_heads
    for name, rows, heads, batch in (("q", args.n, args.heads, args.q_batch), ("k", args.m, Hk, args.kv_batch), ("v", args.m, Hk, args.kv_batch),
                                     ("out", args.n, args.heads, l), ("grad_out", args.n, args.heads, l), ("grad_q", args.n, args.heads, args.q_batch),
                                     ("grad_k", args.m, Hk, args.kv_batch), ("grad_v", args.m, Hk, args.kv_batch),
                                     ("k_prefix", args.prefix, Hk, 1), ("v_prefix", args.prefix, Hk, 1)):
        setattr(args, name, _native.KmHeads(4096, rows * heads * d if batch > 1 else 0, heads * d, d))
    args.lse_stride_l, args.lse_stride_head = args.heads * args.n, args.n
    return args


SCRATCH = [         # sizes, kind; the second and the last two take more than 512 MB
    (dict(l=1, n=1, m=100000, heads=8, key_heads=8, d=128), 0),
    (dict(l=16, q_batch=16, kv_batch=16, n=1024, m=1100, prefix=4000, heads=32, key_heads=8, d=128), 1),
    (dict(l=16, q_batch=16, kv_batch=16, n=1, m=1100, prefix=4000, heads=32, key_heads=8, d=128), 1),
    (dict(l=2, n=3000, m=3500, heads=8, key_heads=8, d=8), 0),
    (dict(l=2, n=3000, m=3500, heads=8, key_heads=8, d=40), 2),
    (dict(l=4, q_batch=4, kv_batch=4, n=64, m=100000, heads=8, key_heads=8, d=128), 2),
    (dict(l=4, q_batch=4, kv_batch=1, n=5000, m=600, heads=32, key_heads=4, d=128), 2),
    (dict(l=64, q_batch=1, kv_batch=64, n=1024, m=200, heads=16, key_heads=16, d=128), 2),
    (dict(l=64, q_batch=64, kv_batch=64, n=2048, m=300, prefix=300, heads=16, key_heads=16, d=64), 1),
]


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("sizes, kind", SCRATCH, ids=str)
def test_scratch_is_what_the_header_says(sizes, kind, dtype):
    args = _big(type=dtype, **sizes)
    l, n, m, H, Hk, d, MB = args.l, args.n, args.m, args.heads, args.key_heads, args.d, 1 << 20
    if kind == 2:
        most = 4 * l * n * H + (dtype == 2) * (4 * l * -(-n // 64) * H + 4 * args.kv_batch * -(-m // 64) * Hk) + 3 * 256 * MB
        if args.q_batch == 1 and l > 1:
            most += 4 * l * n * H * d
    else:
        parts = 8 * l * n * H * (d + 2) if args.prefix and m else 0
        rows = l * n * H + 2 * Hk * (args.kv_batch * m + args.prefix)
        most = max(512 * MB, parts) + (min(384 * rows, 1024 * MB) if dtype == 0 and d <= 64 else 0)
        least = parts
        assert _native.attention_scratch_bytes(args, kind) >= least
    assert 0 <= _native.attention_scratch_bytes(args, kind) <= most + 64
