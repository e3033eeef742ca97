"""Attention of serialised clouds: what runs without a GPU.  Refusals, the tiles
of a ragged batch, the bucket maps and the checks at the C entries."""

from __future__ import annotations

import contextlib
import ctypes

import pytest
import torch
from torch.autograd import forward_ad

from mps_pointops import _native as N
from mps_pointops import attention


def qkv(n=10, m=10, H=4, K=2, D=32, dtype=torch.float32):
    return (torch.zeros(n, H, D, dtype=dtype), torch.zeros(m, K, D, dtype=dtype),
            torch.zeros(m, K, D, dtype=dtype))


OFF = torch.tensor([4, 10])


def call(*tensors, seg=OFF, **kw):
    return attention.window_attention(*tensors, seg, **kw)


def test_cpu_tensors_fail_loudly():
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        call(*qkv())
    q, k, _ = qkv()
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        attention.norm_rotate(q, k, None, None)


def test_attention_refusals():
    q, k, v = qkv()
    with pytest.raises(TypeError, match="torch.Tensor"):
        call([1], k, v)
    with pytest.raises(ValueError, match="shape"):
        call(q[0], k, v)
    with pytest.raises(TypeError, match="float32, float16"):
        call(q.double(), k, v)
    with pytest.raises(TypeError, match="like q"):
        call(q, k.half(), v)
    with pytest.raises(ValueError, match="head size 32"):
        call(q, k[..., :16], v)
    with pytest.raises(ValueError, match="same shape"):
        call(q, k, v[:, :1])
    with pytest.raises(ValueError, match="multiple of 8"):
        call(*(x[..., :12] for x in (q, k, v)))
    with pytest.raises(ValueError, match="multiple of 8"):
        call(*qkv(D=136))
    with pytest.raises(ValueError, match="multiple of k's heads"):
        call(*qkv(H=3, K=2))
    with pytest.raises(ValueError, match=r"\(left, right\)"):
        call(q, k, v, window=5)
    with pytest.raises(ValueError, match="integer"):
        call(q, k, v, window=(1.5, 2))
    with pytest.raises(ValueError, match="sinks"):
        call(q, k, v, sinks=-1)
    with pytest.raises(ValueError, match="scale"):
        call(q, k, v, scale=float("nan"))
    with pytest.raises(ValueError, match="q's row count"):
        call(q, k, v, seg=torch.tensor([4, 9]))
    with pytest.raises(ValueError, match="k's row count"):
        call(q, k, v, seg=attention.Segments(OFF, torch.tensor([4, 12])))


def test_segment_refusals():
    for bad in (torch.tensor([[1]]), torch.tensor([1.0]), [1, 2]):
        with pytest.raises(ValueError, match="one-dimensional"):
            attention.Segments(bad)
    with pytest.raises(ValueError, match="nondecreasing"):
        attention.Segments(torch.tensor([5, 3]))
    with pytest.raises(ValueError, match="nondecreasing"):
        attention.Segments(torch.tensor([-1, 3]))
    with pytest.raises(ValueError, match="batch count"):
        attention.Segments(OFF, torch.tensor([10]))
    with pytest.raises(ValueError, match="2\\^30"):
        attention.Segments(torch.tensor([1 << 30]))


def test_bias_refusals():
    q, k, v = qkv()
    pos = torch.zeros(10, 3, dtype=torch.int32)
    table = torch.zeros(3, 9, 4)
    with pytest.raises(ValueError, match="need a bias_table"):
        call(q, k, v, position=pos)
    with pytest.raises(ValueError, match="position must be an int32"):
        call(q, k, v, bias_table=table)
    with pytest.raises(ValueError, match="position must be an int32"):
        call(q, k, v, bias_table=table, position=pos.float())
    with pytest.raises(ValueError, match=r"shape \(10, 3\)"):
        call(q, k, v, bias_table=table, position=pos[:, :2])
    with pytest.raises(ValueError, match=r"\(A, buckets, 4\)"):
        call(q, k, v, bias_table=table[..., :3], position=pos)
    with pytest.raises(ValueError, match="at most 256"):
        call(q, k, v, bias_table=torch.zeros(3, 87, 4), position=pos)
    with pytest.raises(ValueError, match="2 R \\+ 1"):
        call(q, k, v, bias_table=torch.zeros(3, 8, 4), position=pos)
    with pytest.raises(ValueError, match="2 R \\+ 1"):
        call(q, k, v, bias_table=table, position=pos, buckets=torch.zeros(10, dtype=torch.int32))
    with pytest.raises(ValueError, match="int32"):
        call(q, k, v, bias_table=table, position=pos, buckets=torch.zeros(11))
    q2, k2, v2 = qkv(m=12)
    with pytest.raises(ValueError, match="key_position is needed"):
        call(q2, k2, v2, seg=attention.Segments(OFF, torch.tensor([6, 12])), bias_table=table,
             position=pos)


def test_norm_rotate_refusals():
    q, k, _ = qkv()
    pos, freqs = torch.zeros(10, 1, dtype=torch.int32), torch.zeros(1, 16)

    def refused(match, *args, error=ValueError, **kw):
        with pytest.raises(error, match=match):
            attention.norm_rotate(*args, **kw)

    refused("together", q, k, pos, None)
    refused("row count", q, k[:9], None, None)
    refused("like q", q, k.half(), None, None, error=TypeError)
    refused("multiple of 8", q[..., :12], k[..., :12], None, None)
    refused("float32 or float64", q, k, pos, freqs.half())
    refused("multiple of 4", q, k, pos, torch.zeros(1, 6))
    refused("at most half", q, k, pos, torch.zeros(1, 20))
    refused("1 to 3 axes", q, k, torch.zeros(10, 4, dtype=torch.int32), torch.zeros(4, 16))
    refused("shape", q, k, pos[:4], freqs)
    refused("position must be", q, k, pos.double(), freqs)
    refused("q_weight", q, k, None, None, q_weight=torch.ones(31))
    refused("k_weight", q, k, None, None, k_weight=torch.ones(32, dtype=torch.int32))
    refused("eps", q, k, None, None, eps=-1.0)


def plan(ends, other, keys):
    return attention.Segments._plan(ends, other, keys).tolist()


def test_tiles_cover_each_row_once():
    ends, key_ends = [0, 1, 130, 130, 386], [5, 5, 300, 301, 400]
    tiles = plan(ends, key_ends, 0)
    covered = []
    for row, rows, first, other, lq, lk, base, cloud in tiles:
        assert 1 <= rows <= 128
        start = 0 if cloud == 0 else ends[cloud - 1]
        kstart = 0 if cloud == 0 else key_ends[cloud - 1]
        assert base == start and other == kstart
        assert lq == ends[cloud] - start and lk == key_ends[cloud] - kstart
        assert first == row - start + lk - lq
        covered += range(row, row + rows)
    assert covered == list(range(386))
    covered, order = [], []
    for row, rows, first, other, lq, lk, base, cloud in plan(key_ends, ends, 1):
        assert first == row - base
        covered += range(row, row + rows)
        order.append((first, cloud))
    assert sorted(covered) == list(range(400))
    assert order == sorted(order)  # first tiles of all clouds, then second ones
    assert plan([], [], 0) == []


def test_segments_on_cpu():
    seg = attention.Segments(torch.tensor([3, 3, 200]), torch.tensor([3, 8, 500]))
    assert (seg.clouds, seg.rows, seg.keys, seg.max_rows, seg.max_keys) == (3, 200, 500, 197, 492)
    empty = attention.Segments(torch.zeros(0, dtype=torch.int64))
    assert (empty.clouds, empty.rows, empty.max_rows) == (0, 0, 0)


def test_log_buckets():
    m = attention.log_buckets(8, 16, bidirectional=False)
    assert m.dtype == torch.int32 and m.numel() == 33
    at = lambda d: int(m[d + 16])  # noqa: E731
    assert [at(d) for d in (5, 0, -1, -2, -3)] == [0, 0, 1, 2, 3]
    # 4 + floor(4 log(n / 4) / log(4)): 4..5 -> 4, 6..7 -> 5, 8..11 -> 6, 12.. -> 7
    assert [at(-n) for n in (4, 5, 6, 7, 8, 11, 12, 15, 16)] == [4, 4, 5, 5, 6, 6, 7, 7, 7]
    b = attention.log_buckets(8, 16)
    assert int(b[16]) == 0 and int(b[15]) == 1 and int(b[17]) == 5
    assert b.max() == 7 and b.min() == 0
    for bad in ((2, 16, True), (8, 0, True), (8, 2, True), (8, 5000, True)):
        with pytest.raises(ValueError):
            attention.log_buckets(*bad)


def test_c_entries_validate_before_device_work():
    lib = N.lib()
    a = N.AttentionArgs(heads=4, kv_heads=3, dim=32, scale=1.0)
    assert lib.mpo_window_attention(ctypes.byref(a), None) == 1
    assert "multiple of kv_heads" in N.last_error()
    a = N.AttentionArgs(heads=4, kv_heads=2, dim=20, scale=1.0)
    assert lib.mpo_window_attention(ctypes.byref(a), None) == 1 and "multiple of 8" in N.last_error()
    a = N.AttentionArgs(heads=4, kv_heads=2, dim=32, scale=1.0, table=16, axes=3, buckets=100)
    assert lib.mpo_window_attention(ctypes.byref(a), None) == 1 and "256" in N.last_error()
    a = N.AttentionArgs(heads=4, kv_heads=2, dim=32, scale=1.0, q_tile_count=1)
    assert lib.mpo_window_attention(ctypes.byref(a), None) == 1 and "null" in N.last_error()
    assert lib.mpo_window_attention(None, None) == 1
    assert lib.mpo_window_attention_backward(None, None) == 1
    a = N.AttentionArgs(heads=4, kv_heads=2, dim=32, scale=1.0)
    assert lib.mpo_window_attention(ctypes.byref(a), None) == 0  # nothing to do
    r = N.RotateArgs(heads=2, kv_heads=2, dim=32, pairs=6, axes=1)
    assert lib.mpo_norm_rotate(ctypes.byref(r), None) == 1 and "pairs" in N.last_error()
    r = N.RotateArgs(heads=2, kv_heads=2, dim=32, rows=3)
    assert lib.mpo_norm_rotate(ctypes.byref(r), None) == 1 and "null" in N.last_error()
    assert lib.mpo_norm_rotate(None, None) == 1


def test_argument_blocks_match_the_header(tmp_path):
    """Sizes and the last members' offsets of the structures, by the C compiler."""
    import shutil
    import subprocess

    from conftest import ROOT

    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include "mpo_b200.h"\nint main(void){printf("%zu %zu %zu '
                   '%zu %zu\\n", sizeof(mpo_rotate), offsetof(mpo_rotate, eps), '
                   'sizeof(mpo_attention), offsetof(mpo_attention, workspace), '
                   'offsetof(mpo_attention, scale));return 0;}\n')
    subprocess.run([cc, "-I", str(ROOT / "include"), str(src), "-o", str(tmp_path / "sizes")],
                   check=True)
    out = subprocess.run([str(tmp_path / "sizes")], check=True, capture_output=True, text=True)
    want = [ctypes.sizeof(N.RotateArgs), N.RotateArgs.eps.offset, ctypes.sizeof(N.AttentionArgs),
            N.AttentionArgs.workspace.offset, N.AttentionArgs.scale.offset]
    assert [int(x) for x in out.stdout.split()] == want


def test_entry_addresses_of_the_tensor_core_kernels():
    """The kernels form the address of a pair's table entry by two float32
    multiply-adds, t = sat(column / 2R + part) and t * 256 R + first in denormals.
    Their roundings leave every address exact for rows within 2^15 of the tile's
    first and columns clamped at 2^16 (float64 carries the products exactly)."""
    import numpy as np

    f = np.float32
    rng = np.random.default_rng(0)
    for reach in [0, 1, 2, 3, 7, 15, 31, 42, 63, 127, 128, 500, 1023, 1024]:
        inv = f(1) / f(2 * reach) if reach else f(0)
        d = np.concatenate([np.arange(-reach - 2, reach + 3), [-65536, 65536, -40000, 40000]])
        for row in [0, 1, -1, 32768, -32768, 32767, *rng.integers(-32768, 32769, 200)]:
            part = f(0.5 - float(row) * float(inv))
            column = np.clip(d + row, -65536, 65536)
            t = np.clip((column * float(inv) + float(part)).astype(f), f(0), f(1))
            for first in (1028, 200004):
                address = np.rint(t.astype(np.float64) * (256 * reach) + first)
                want = first + 128 * (np.clip(column - row, -reach, reach) + reach)
                assert (address == want).all(), (reach, row)


@pytest.fixture
def recorder(monkeypatch):
    """The native calls replaced by ones that note their arguments and leave zeros, so
    that what the Python side does runs on CPU tensors."""
    calls = []

    def attention_call(backward, *args):
        calls.append((backward, args))
        for x in args[-4:] if backward else args[-2:]:  # dq, dk, dv, dtable; out, lse
            if x is not None:
                x.zero_()

    monkeypatch.setattr(N, "require_cuda", lambda t, what: None)
    monkeypatch.setattr(attention, "_attention_call", attention_call)
    return calls


@pytest.mark.parametrize("which", ["position", "key_position", "buckets"])
def test_positions_changed_before_the_backward_are_refused(recorder, which):
    """The backward forms the bias again: a position or map that the caller has
    refilled since the forward is an error, as it is for every other saved input."""
    q, k, v = (x.requires_grad_() for x in qkv())
    kw = dict(position=torch.zeros(10, 1, dtype=torch.int32),
              key_position=torch.zeros(10, 1, dtype=torch.int32),
              buckets=torch.zeros(9, dtype=torch.int32))
    out = call(q, k, v, bias_table=torch.zeros(1, 5, 4), **kw)
    out.sum().backward(retain_graph=True)
    assert [backward for backward, _ in recorder] == [False, True]
    kw[which].fill_(3)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


def test_long_positions_reach_the_kernel_whole(monkeypatch):
    """int64 positions go to norm_rotate's kernel as they are, not cut to 32 bits."""
    seen = {}

    def pack(*values):
        args = dict(zip((name for name, _ in N.RotateArgs._fields_), values))
        kind = {0: ctypes.c_int32, 1: ctypes.c_float, 2: ctypes.c_int64}[args["position_float"]]
        seen["position"] = list((kind * 10).from_address(args["position"]))
        return b""

    class Library:
        def mpo_norm_rotate(self, args, stream):
            return 0

    monkeypatch.setattr(N, "require_cuda", lambda t, what: None)
    monkeypatch.setattr(N, "lib", Library)
    monkeypatch.setattr(N, "on_device", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(attention, "_pack_rotate", pack)
    monkeypatch.setattr(attention, "_stream", lambda device: 0)
    q, k, _ = qkv()
    want = [(1 << 32) + 3, -(1 << 40), 7, *range(7)]
    attention.norm_rotate(q, k, torch.tensor(want), torch.zeros(1, 16, dtype=torch.float64))
    assert seen["position"] == want


def test_c_entry_refuses_position_types_and_addresses():
    lib = N.lib()
    for bad, match in ((dict(position_float=3), "position type"), (dict(position_float=-1), "position type"),
                       (dict(position_float=2, position=36), "aligned"), (dict(position=34), "aligned")):
        args = dict(q=16, k=16, out_q=16, out_k=16, position=32, freqs=32, rows=3, heads=2, kv_heads=2, dim=32,
                    pairs=8, axes=1)
        r = N.RotateArgs(**{**args, **bad})
        assert lib.mpo_norm_rotate(ctypes.byref(r), None) == 1 and match in N.last_error()


def test_long_positions_of_the_bias_clamp(recorder):
    """int64 positions beyond the kernels' range end at its limits, they do not wrap."""
    far = torch.tensor([0, 5, (1 << 32) + 3, -(1 << 32) - 3, (1 << 31), 1 << 62, -(1 << 63), (1 << 30) - 1, -7, 1])
    call(*qkv(), bias_table=torch.zeros(1, 5, 4), position=far, key_position=far.flip(0))
    top = (1 << 30) - 1
    want = [0, 5, top, -top, top, top, -top, top, -7, 1]
    _, (_, _, _, _, (_, qpos, kpos, _), *_) = recorder[0]
    assert qpos.dtype == kpos.dtype == torch.int32
    assert qpos[:, 0].tolist() == want and kpos[:, 0].tolist() == want[::-1]


@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_derivatives_are_refused(recorder, monkeypatch, grad):
    """No forward-mode formula: a tangent is an error, not lost, where no input requires
    a gradient and where gradients are off."""
    def rotate_call(backward, q, k, wq, wk, position, freqs, eps, interleaved, out_q, out_k, *_):
        out_q.zero_()
        out_k.zero_()

    monkeypatch.setattr(attention, "_rotate_call", rotate_call)
    q, k, v = qkv()
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        dual = forward_ad.make_dual(k, torch.ones_like(k))
        with pytest.raises(RuntimeError, match="forward mode AD"):
            call(q, dual, v)
        with pytest.raises(RuntimeError, match="forward mode AD"):
            attention.norm_rotate(q, dual, None, None)
        weight = forward_ad.make_dual(torch.ones(32), torch.ones(32))
        with pytest.raises(RuntimeError, match="forward mode AD"):
            attention.norm_rotate(q, k, None, None, k_weight=weight)
        table = forward_ad.make_dual(torch.zeros(1, 5, 4), torch.ones(1, 5, 4))
        with pytest.raises(RuntimeError, match="forward mode AD"):
            call(q, k, v, bias_table=table, position=torch.zeros(10, dtype=torch.int32))


def test_calls_without_gradients_keep_nothing(recorder):
    q, k, v = qkv()
    out = call(q, k, v)
    assert out.grad_fn is None and not out.requires_grad
    out, lse = call(q, k, v, return_lse=True)
    assert lse.shape == (4, 10) and lse.grad_fn is None
    q.requires_grad_()
    with torch.no_grad():
        out = call(q, k, v)
    assert out.grad_fn is None
    with torch.inference_mode():
        assert call(q, k, v).is_inference()
    assert [args[6] is None for _, args in recorder] == [True, False, True, True]  # lse only where it is used


def test_waits_that_ran_out_are_reported_to_their_stream(monkeypatch):
    """The word that a kernel sets belongs to its stream: the next call there is told, once;
    calls on other streams are not, and check() is told without a further call."""
    first, second = torch.device("cuda", 0), torch.device("cuda", 1)
    words = {key: ctypes.c_int32(0) for key in ((0, 16), (0, 32), (1, 16))}
    monkeypatch.setattr(attention, "_statuses", {key: (None, word) for key, word in words.items()})
    monkeypatch.setattr(torch.cuda, "synchronize", lambda device=None: None)
    words[0, 16].value = 1
    for device, stream in ((first, 32), (second, 16)):
        assert attention._status(device, stream) == ctypes.addressof(words[device.index, stream])
    with pytest.raises(RuntimeError, match="ran out"):
        attention._status(first, 16)
    assert attention._status(first, 16) == ctypes.addressof(words[0, 16])
    words[0, 32].value = 1
    attention.check(second)
    with pytest.raises(RuntimeError, match="ran out"):
        attention.check(first)
    attention.check(first)
    words[0, 16].value = words[0, 32].value = 1
    with pytest.raises(RuntimeError, match="ran out"):
        attention.check("cuda:0")
    assert attention._status(first, 16) and attention._status(first, 32)  # both words were read


def test_entry_addresses_for_every_reach():
    """As above for each reach that a table or a bucket map can have: rows at the ends of
    their range and beside the tile's first, differences around the clamps and at random."""
    import numpy as np

    f = np.float32
    rng = np.random.default_rng(1)
    rows = np.array([0, 1, -1, 5, 32767, 32768, -32767, -32768, *rng.integers(-32768, 32769, 24)])[:, None]
    for reach in range(attention._MAX_REACH + 1):
        inv = f(1) / f(2 * reach) if reach else f(0)
        d = np.unique(np.concatenate([np.arange(-3, 4), reach + np.arange(-3, 3), -reach + np.arange(-2, 4),
                                      rng.integers(-reach - 1, reach + 2, 40), [-98304, 98304]]))[None]
        part = (0.5 - rows * float(inv)).astype(f)
        column = np.clip(d + rows, -65536, 65536)
        t = np.clip((column * float(inv) + part.astype(np.float64)).astype(f), f(0), f(1))
        want = 128 * (np.clip(column - rows, -reach, reach) + reach)
        for first in (1028, 200004):
            assert (np.rint(t.astype(np.float64) * (256 * reach) + first) == first + want).all(), reach
