"""The paged key-value cache at its edges: settings in which nothing is chosen, values that few bits lose, calls that
follow each other without a pause, ids of 64 bits, caches that share memory.

The oracles are those of test_paged_cache.py: the operators' definition in 64 bits, position by position.
"""
import os
import re
import subprocess
import sys
import threading
import time

import numpy as np
import pytest
import torch

from conftest import ROOT
from test_paged_cache import DT, dev, make_case, np64, oracle_evict


# ------------------------------------------------------------------------------------------------ eviction
@pytest.mark.gpu
@pytest.mark.parametrize("lens,page,init,local", [
    ([131072, 130999], 1, 64, 4096), ([300, 301, 5000, 0, 1], 1, 4, 6), ([409600], 1, 0, 1), ([65536, 100, 40000], 16, 1, 63),
    ([9000] * 70, 64, 3, 8), ([2000] * 300, 16, 0, 5)])
def test_eviction_to_the_first_and_last_pages(lens, page, init, local):
    """A budget that the first and the last pages fill: nothing is chosen, whatever the weights are and whatever the kernel
    before left on the chip (here all bits set, from a cache that is full of them)."""
    from unum_ops_b200 import evict_cache, paged_attention

    d = dev()
    rng = np.random.default_rng(len(lens) + lens[0])
    width = min(max(-(-n // page) for n in lens) + 1, 409600)
    table = rng.permutation(len(lens) * width).reshape(len(lens), width).astype(np.int32)
    w = rng.standard_normal((len(lens), 2, width * page)).astype(np.float32)
    w[..., ::7] = np.nan
    ln = np.array(lens, np.int32)
    args = [torch.from_numpy(x).to(d) for x in (table, ln, w)]
    want = oracle_evict(table, ln, w, init + local, init, local, page)
    q, kc, _, rows, n = [x.to(d) for x in make_case(3, [60000, 60000], 2, 16, 128, 1, "bf16")]
    kc.view(torch.int16).fill_(-1)
    for _ in range(10):
        paged_attention(q, kc, kc, rows, n)
        got = evict_cache(*args, budget=init + local, init_pages=init, local_pages=local, page_size=page)
        for name, x, y in zip(("table", "seqlens", "weights", "evicted"), got, want):
            np.testing.assert_array_equal(x.cpu().numpy(), y, err_msg=name)


# ------------------------------------------------------------------------------------------------ values that few bits lose
# The kernels hold a probability in the cache's type as 2^(s - m + lift), m a maximum of the scores (base 2) of the warp's
# positions and lift 12 in fp16.  A rounding is off by eps/2 of the probability, or where that is subnormal by half of the
# smallest subnormal: 2^-25 in fp16, 2^-37 of the largest probability.  The sum of all is at least the largest, so
#     |err| <= eps/2 * (|out| + sum p|v|) + 2^-16 * sum p|v| + 2^-37 * sum |v| + 2^-25 (fp16's subnormal outputs)
# with the scores exact here (one product each).  In bf16, whose exponents are fp32's, the last two are 0.
@pytest.mark.gpu
@pytest.mark.parametrize("gap", [0, 10, 14, 17, 18, 24])
@pytest.mark.parametrize("n,Hk,G,D,at,spread", [(16, 1, 1, 64, 0, 0), (700, 2, 16, 128, 0, 1), (16384, 1, 16, 128, 0, 0), (16384, 2, 4, 64, 9000, 1),
                                                (40000, 2, 16, 128, 39999, 1), (9000, 1, 33, 64, 4, 0), (131072, 1, 16, 128, 0, 1)])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_one_key_far_above_the_others(dtype, n, Hk, G, D, at, spread, gap):
    """An attention sink: one key `gap` nats above the others' mean, its value 0.  The others are the output."""
    from unum_ops_b200 import paged_attention

    rng = np.random.default_rng(n + G)
    t = lambda x: torch.from_numpy(x.astype(np.float32)).to(DT[dtype])  # noqa: E731
    q, k = np.zeros((1, Hk * G, D)), np.zeros((n, Hk, D))
    q[:, :, 0], k[:, :, 0] = 1, spread * rng.standard_normal((n, Hk))
    k[at, :, 0] = gap
    v = rng.uniform(0.5, 8, (n, Hk, D))
    v[at] = 0
    q, k, v = t(q), t(k), t(v)
    d = dev()
    out = np64(paged_attention(q.to(d), k.to(d), v.to(d), torch.arange(n, dtype=torch.int32, device=d)[None],
                               torch.tensor([n], dtype=torch.int32, device=d), softmax_scale=1.0))[0].reshape(Hk, G, D)
    s = np64(k)[:, :, 0]
    p = np.exp(s - s.max(0))
    p /= p.sum(0)
    ref = np.einsum("nh,nhd->hd", p, np64(v))[:, None]  # the values are positive: sum p|v| as well
    small = 2.0 ** -37 * np64(v).sum(0)[:, None] + 2.0 ** -25 if dtype == "fp16" else 0
    allow = 2 * torch.finfo(DT[dtype]).eps / 2 * ref + 2.0 ** -16 * ref + small
    err = np.abs(out - ref)
    assert np.all(err <= allow), f"off by {np.max(err / allow)} of what is allowed"


@pytest.mark.gpu
@pytest.mark.parametrize("n,G", [(1000, 16), (1000, 32), (40000, 16)])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_scores_of_any_magnitude(dtype, n, G):
    """Scores from 1 to 2^31, a few of their last places apart: their maximum is taken out without what it is shifted by
    being rounded into an overflow.  All values are 1, and so is the output, to a rounding of each probability and one of
    the output."""
    from unum_ops_b200 import paged_attention

    d = dev()
    rng = np.random.default_rng(n)
    heads = 2 * G
    q, k = torch.zeros(1, heads, 64), torch.zeros(n, 2, 64)
    q[..., 0] = 32768.0
    q[..., 1] = torch.from_numpy(np.exp2(rng.integers(0, 8, heads)))
    k[..., 1] = torch.from_numpy(rng.uniform(0, 30, (n, 2)))
    v = torch.ones(n, 2, 64, dtype=DT[dtype], device=d)
    table, ln = torch.arange(n, dtype=torch.int32, device=d)[None], torch.tensor([n], dtype=torch.int32, device=d)
    for e in range(-15, 16):
        for sign in (1, -1):
            k[..., 0] = sign * 2.0 ** e * torch.from_numpy(rng.uniform(1, 1.001 if e < 4 else 1, (n, 2)))
            out = paged_attention(q.to(DT[dtype]).to(d), k.to(DT[dtype]).to(d), v, table, ln, softmax_scale=1.0).double()
            err = float((out - 1).abs().nan_to_num(nan=float("inf")).max())
            assert err <= torch.finfo(DT[dtype]).eps + 2.0 ** -16, (e, sign, err)


# ------------------------------------------------------------------------------------------------ barriers
def test_warps_come_together_before_the_barriers_that_ask_for_it():
    """A cluster's barrier (.aligned) and bar.sync are for whole warps: in the paged cache's kernels and in what they share
    with others, a __syncwarp stands before each."""
    csrc, found = os.path.join(ROOT, "unum_ops_b200", "csrc"), 0
    for name in ("paged_attention.cu", "paged_cache.cu", "sm100.cuh"):
        with open(os.path.join(csrc, name)) as f:
            text = re.sub(r"//[^\n]*", "", f.read())
        for m in re.finditer(r"(if \([^)]*\)\s*|else\s*)?asm volatile\(\s*\"(barrier\.cluster\.\w+|bar\.sync)", text):
            if name == "sm100.cuh" and m.group(2) == "bar.sync":
                continue  # its callers' business: no paged kernel is one
            found += 1
            assert text[:m.start()].rstrip().endswith("__syncwarp();"), (name, m.group(0))
        assert not re.search(r"\.aligned;\\n\\t *barrier", text), name
    assert found >= 3


# ------------------------------------------------------------------------------------------------ calls without a pause
def test_kernels_that_start_early_read_nothing_through_the_read_only_path():
    """A kernel that is launched behind one that still runs may not use loads for memory that never changes."""
    csrc, found = os.path.join(ROOT, "unum_ops_b200", "csrc"), 0
    for name in sorted(os.listdir(csrc)):
        with open(os.path.join(csrc, name)) as f:
            text = re.sub(r"//[^\n]*", "", f.read())
        if name.endswith(".cu") and "wait_for_previous_kernel" in text:
            found += 1
            assert not re.search(r"__ldg|__restrict__|ld\.global\.nc", text), name
    assert found >= 2


@pytest.mark.gpu
@pytest.mark.parametrize("lens,new", [([500, 41, 1, 177], [3, 1, 1, 100]), ([30001, 40, 300, 17771], [900, 1, 299, 5]), ([900] * 150, [1] * 150)])
@pytest.mark.parametrize("graph", [False, True])
def test_a_step_of_all_operators_without_a_pause(lens, new, graph):
    """Writes, attention that gathers weights, eviction by them and attention over what is left, launched one right behind
    the other (every argument is as the kernels take it, so that nothing lies between), give the bits that the same calls
    give with a pause after each.  The buffers are the same in every turn and hold other values each time."""
    from unum_ops_b200 import append_cache, evict_cache, paged_attention

    d, B, T = dev(), len(lens), sum(new)
    q, kc, vc, table, ln = [x.to(d) for x in make_case(5, lens, 2, 16, 128, 1, "bf16", spare=1 + max(lens) % 2)]
    W = table.shape[1]
    assert W % 2 == 1
    bs = torch.repeat_interleave(torch.arange(B), torch.tensor(new)).to(torch.int32).to(d)
    pos = torch.cat([torch.arange(n - m, n) + 1 for n, m in zip(lens, new)]).to(torch.int32).to(d)
    k, v, w = *torch.zeros(2, T, 2, 128, dtype=torch.bfloat16, device=d), torch.zeros(B, 2, W, device=d)

    def step(pause):
        append_cache(k, v, kc, vc, table, bs, pos)
        pause()
        a = paged_attention(q, kc, vc, table, ln, weights=w, return_lse=True)
        pause()
        e = evict_cache(table, ln, w, budget=33, init_pages=1, local_pages=3)
        pause()
        b = paged_attention(q, kc, vc, e[0], e[1], weights=e[2], return_lse=True)
        pause()
        return [*a, *e, *b]

    start = [x.clone() for x in (kc, vc)]
    g = torch.Generator(device=d).manual_seed(1)
    if graph:
        step(torch.cuda.synchronize)
        captured = torch.cuda.CUDAGraph()
        with torch.cuda.graph(captured):
            outs = step(lambda: None)
    for turn in range(12):
        values = [torch.randn(x.shape, generator=g, device=d).to(x.dtype) for x in (q, k, v)] + [torch.rand(w.shape, generator=g, device=d)]
        got = []
        for pause in (torch.cuda.synchronize, lambda: None):
            kc.copy_(start[0]), vc.copy_(start[1])
            for x, y in zip((q, k, v, w), values):
                x.copy_(y)
            torch.cuda.synchronize()
            if graph and got:
                captured.replay()
                res = outs
            else:
                res = step(pause)
            torch.cuda.synchronize()
            got.append([x.clone() for x in (*res, kc, vc, w)])
        assert all(torch.equal(x, y) for x, y in zip(*got)), turn


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[500, 41, 0, 177], [30000, 40, 300, 17771]])
@pytest.mark.parametrize("graph", [False, True])
def test_two_streams_that_part_and_meet(lens, graph):
    """Copies into the inputs, a write, attention on two streams at once, and eviction on the first by what the other has
    gathered: eager, and as one graph with a fork and a join."""
    from unum_ops_b200 import append_cache, evict_cache, paged_attention

    d = dev()
    q, kc, vc, table, ln = [x.to(d) for x in make_case(6, lens, 2, 16, 128, 1, "bf16")]
    W = table.shape[1]
    qs, qs_in, ws = [torch.empty_like(q) for _ in range(2)], [torch.empty_like(q) for _ in range(2)], [torch.zeros(4, 2, W, device=d) for _ in range(2)]
    k, bs = torch.randn(4, 2, 128, device=d).to(torch.bfloat16), torch.arange(4, dtype=torch.int32, device=d)
    side, g = torch.cuda.Stream(), torch.Generator(device=d).manual_seed(3)

    def step(other):
        for x, y, w in zip(qs, qs_in, ws):
            x.copy_(y)
            w.zero_()
        append_cache(k, k, kc, vc, table, bs, ln)
        main = torch.cuda.current_stream()
        if other:
            other.wait_stream(main)
        with torch.cuda.stream(other or main):
            a = paged_attention(qs[0], kc, vc, table, ln, weights=ws[0], return_lse=True)
        b = paged_attention(qs[1], kc, vc, table, ln, weights=ws[1], return_lse=True)
        if other:
            main.wait_stream(other)
        e = evict_cache(table, ln, ws[0], budget=30)
        c = paged_attention(qs[0], kc, vc, e[0], e[1], weights=ws[1], return_lse=True)
        return [*a, *b, *e, *c, *ws]

    if graph:
        step(None)
        torch.cuda.synchronize()
        captured = torch.cuda.CUDAGraph()
        with torch.cuda.graph(captured):
            outs = step(side)
    for _ in range(10):
        for x in qs_in:
            x.copy_(torch.randn(x.shape, generator=g, device=d))
        torch.cuda.synchronize()
        want = [x.clone() for x in step(None)]
        torch.cuda.synchronize()
        if graph:
            captured.replay()
        else:
            outs = step(side)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(outs, want))


# ------------------------------------------------------------------------------------------------ ids that 32 bits do not hold
WIDE = [(torch.int64, 1 << 32), (torch.int64, -(1 << 32)), (torch.int64, 3 << 40), (torch.uint32, 3 << 30), (torch.uint64, 1 << 63), (torch.float64, 2.0 ** 40),
        (torch.float64, float("inf")), (torch.float32, float("nan"))]


def widened(x, dtype, at, value):
    """x in another type, with a value at one place."""
    x = x.to(torch.float64 if dtype.is_floating_point else torch.int64).clone()
    if dtype in (torch.uint32, torch.uint64):
        x = x.clamp(min=0)
        value = value - (1 << 64) if value >= 1 << 63 else value
    x[at] = value
    return x.view(dtype) if dtype == torch.uint64 else x.to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,value", WIDE)
def test_ids_that_32_bits_do_not_hold(dtype, value):
    """Wider integers and floating-point numbers are taken where int32 is asked for; what is out of its range is out of the
    table's, the cache's and the batch's too, and a length above the bound is cut to the bound."""
    from unum_ops_b200 import append_cache, evict_cache, paged_attention

    d, lens = dev(), [40, 25]
    q, kc, vc, table, ln = [x.to(d) for x in make_case(8, lens, 2, 4, 64, 1, "bf16")]
    table[0, 9] = table[0, 0]
    table[0, 0], table[0, 30:35], table[1, 25:] = 0, 1, 0
    hidden = table.clone()
    hidden[0, 9] = -1
    wide = widened(table, dtype, (0, 9), value)
    assert torch.equal(paged_attention(q, kc, vc, wide, ln), paged_attention(q, kc, vc, hidden, ln))
    top, no_number = value > 0, value != value
    clamped = ln.clone()
    clamped[1] = table.shape[1] if top and not no_number else 0
    long = widened(ln, dtype, 1, value)
    assert torch.equal(paged_attention(q, kc, vc, table, long), paged_attention(q, kc, vc, table, clamped))
    w = torch.rand(2, 2, table.shape[1], device=d)
    assert all(torch.equal(x, y) for x, y in zip(evict_cache(table, long, w, budget=20), evict_cache(table, clamped, w, budget=20)))
    k = torch.randn(3, 2, 64, device=d).to(torch.bfloat16)
    bs, pos = torch.tensor([0, 0, 1], device=d), torch.tensor([1, 10, 3], device=d)
    want = kc.clone()
    want[table[0, 0].long()], want[table[1, 2].long()] = k[0], k[2]
    for args in ((wide, bs, pos), (table, widened(bs, dtype, 1, value), pos), (table, bs, widened(pos, dtype, 1, value))):
        a, b = kc.clone(), vc.clone()
        append_cache(k, k, a, b, *args)
        assert torch.equal(a, want)


@pytest.mark.gpu
def test_a_position_past_32_bits_in_a_table_that_reaches_so_far():
    """A table of 2^31 positions and more: positions from 2^31 - 2 on are outside."""
    from unum_ops_b200 import append_cache

    d = dev()
    kc, vc = torch.zeros(2, 65536, 1, 64, device=d, dtype=torch.bfloat16)
    table = torch.full((1, 1 << 16), -1, device=d, dtype=torch.int32)
    table[0, (1 << 15) - 1] = 0  # the page that ends at 2^31
    k = torch.ones(3, 1, 64, device=d, dtype=torch.bfloat16)
    pos = torch.tensor([(1 << 31) - 2, 1 << 31, 1 << 40], device=d)
    append_cache(k, k, kc, vc, table, torch.zeros(3, dtype=torch.int32, device=d), pos, page_size=65536)
    want = torch.zeros(65536, device=d)
    want[65536 - 3] = 1
    assert torch.equal(kc[:, 0, 0].float(), want) and torch.equal(vc, kc)


# ------------------------------------------------------------------------------------------------ caches that share memory
def cache_pairs():
    """(k_cache, v_cache, whether they share memory) in one buffer each."""
    D = 64
    t = lambda *s: torch.zeros(s, dtype=torch.bfloat16)  # noqa: E731
    b = t(13, 3, D)
    yield b[:12], b[1:], True                                   # a token apart
    yield b[:, :2], b[:, 1:], True                              # a head apart
    yield b[:, :1], b[:, 1:2], False                            # heads side by side
    yield b[:, ::2], b[:, 1:2].expand(13, 2, D)[:, :2], True    # an expanded one
    c = t(13, 2, 2, D)
    yield c[:, 0], c[:, 1], False                               # interleaved token by token
    yield c[:12, 0], c[1:, 0], True
    yield c[:12, 1], c[1:, 0], False                            # a token apart, interleaved all the same
    yield c[:, :, 0], c[:, :, 1], False                         # interleaved head by head
    yield c[:, :, 0], c[:, 1], True
    yield c[:6, 0], c[7:, 0][:6], False                         # one behind the other
    e = t(13, 6, D)
    yield e[:, :4:2], e[:, 1:3], True                           # heads 0, 2 and 1, 2
    yield e[:, :4:2], e[:, 1::4], False                         # heads 0, 2 and 1, 5: different strides
    f = t(4 * 13 * D)
    yield f[:].as_strided((13, 2, D), (4 * D, D, 1)), f.as_strided((13, 2, D), (4 * D, D, 1), D // 2), True   # half a row apart
    yield f.as_strided((13, 2, D), (4 * D, D, 1)), f.as_strided((13, 2, D), (4 * D, D, 1), 2 * D - 8), True   # by its last piece
    yield f.as_strided((12, 2, D), (4 * D, D, 1)), f.as_strided((12, 2, D), (4 * D, D, 1), 6 * D), False
    yield f.as_strided((12, 2, D), (4 * D, D, 1)), f.as_strided((12, 2, D), (2 * D, D, 1), 2 * D), True       # strides of their own
    yield t(1, 2, D), t(1, 2, D), False
    g = t(3, D)
    yield g[None, :2], g[None, 1:], True                        # a cache of one token
    yield t(0, 2, D), t(0, 2, D), False


@pytest.mark.parametrize("i", range(len(list(cache_pairs()))))
def test_caches_that_share_memory_are_refused(i):
    from unum_ops_b200 import append_cache

    k, v, shared = list(cache_pairs())[i]
    new, ids = torch.zeros(2, k.shape[1], 64, dtype=torch.bfloat16), torch.ones(2, dtype=torch.int32)
    table = torch.zeros(2, 12, dtype=torch.int32)
    for a, b in ((k, v), (v, k)):
        with pytest.raises(ValueError, match="share memory" if shared else "CUDA"):  # these are on the CPU
            append_cache(new, new, a, b, table, ids, ids)
        # as the rows' addresses have it
        rows = [{x.data_ptr() + 2 * (i * x.stride(0) + h * x.stride(1) + d) for i in range(x.shape[0]) for h in range(x.shape[1])
                 for d in range(64)} for x in (a, b)]
        expanded = any(len(r) < x.numel() for r, x in zip(rows, (a, b)))
        assert shared == (expanded or bool(rows[0] & rows[1]))


# ------------------------------------------------------------------------------------------------ refusals
@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("which", ["q", "kc", "vc", "w", "k", "v"])
def test_tangents_are_refused(which, grad):
    """Dual tensors of forward mode, under torch.no_grad() too, which does not turn that mode off."""
    import torch.autograd.forward_ad as fwd

    from unum_ops_b200 import append_cache, evict_cache, paged_attention

    q, kc, vc, table, ln = make_case(1, [5, 9], 2, 4, 64, 1, "bf16")
    x = dict(q=q, kc=kc, vc=vc, w=torch.zeros(2, 2, table.shape[1]), k=kc[:2].clone(), v=vc[:2].clone())
    with fwd.dual_level(), torch.set_grad_enabled(grad):
        x[which] = fwd.make_dual(x[which], torch.ones_like(x[which]))
        calls = [lambda: paged_attention(x["q"], x["kc"], x["vc"], table, ln, weights=x["w"])] if which not in "kv" else []
        if which == "w":
            calls.append(lambda: evict_cache(table, ln, x["w"], budget=4))
        if which not in "qw":
            calls.append(lambda: append_cache(x["k"], x["v"], x["kc"], x["vc"], table, ln, ln))
        for call in calls:
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()


def test_a_return_lse_without_a_truth_value_raises_its_own_error():
    from unum_ops_b200 import paged_attention

    class NoTruth:
        def __bool__(self):
            raise ZeroDivisionError("no truth")

    q, kc, vc, table, ln = make_case(1, [5, 9], 2, 4, 64, 1, "bf16")
    with pytest.raises(ZeroDivisionError, match="no truth"):
        paged_attention(q, kc, vc, table, ln, return_lse=NoTruth())
    with pytest.raises(RuntimeError, match="ambiguous"):
        paged_attention(q, kc, vc, table, ln, return_lse=torch.zeros(2))


# ------------------------------------------------------------------------------------------------ the build
def test_the_binding_is_built_again_for_another_torch_or_python(monkeypatch):
    """It is bound to torch's C++ ABI and to Python's: one compiled for others is neither current nor loaded."""
    import sysconfig

    from unum_ops_b200 import _build, _lib

    _build.build()
    assert not _build.needs_build()
    for where, name, value in ((torch, "__version__", "2.99.0"), (sysconfig, "get_config_var", lambda _: "cpython-399")):
        with monkeypatch.context() as m:
            m.setattr(where, name, value)
            assert _build.needs_build()
            m.setattr(_lib, "_native", None)
            with pytest.raises(RuntimeError, match="build it"):
                _lib.binding()
    assert not _build.needs_build()


# ------------------------------------------------------------------------------------------------ other threads
@pytest.mark.gpu
@pytest.mark.parametrize("op", ["append", "attend", "evict"])
def test_other_threads_run_while_a_call_waits_for_the_device(op):
    """A launch waits where the device's queue of launches is full (here behind a kernel that takes most of a second).
    Python's other threads run meanwhile."""
    from unum_ops_b200 import append_cache, evict_cache, paged_attention

    q, kc, vc, table, ln = [x.to(dev()) for x in make_case(1, [5, 9], 2, 4, 64, 1, "bf16")]
    k, w = kc[:2].clone(), torch.zeros(2, 2, table.shape[1], device=dev())
    call = {"append": lambda: append_cache(k, k, kc, vc, table, ln, ln), "attend": lambda: paged_attention(q, kc, vc, table, ln),
            "evict": lambda: evict_cache(table, ln, w, budget=4)}[op]
    for _ in range(3):
        call()
    torch.cuda.synchronize()
    ticks, done = [], threading.Event()

    def tick():
        while not done.is_set():
            ticks.append(time.perf_counter())
            time.sleep(0.002)

    other = threading.Thread(target=tick)
    other.start()
    begin = time.perf_counter()
    torch.cuda._sleep(1_500_000_000)
    longest = 0.0
    for _ in range(3000):
        t = time.perf_counter()
        call()
        longest = max(longest, time.perf_counter() - t)
    torch.cuda.synchronize()
    end = time.perf_counter()
    done.set()
    other.join()
    ticks = [begin] + [t for t in ticks if begin < t < end] + [end]
    pause = max(b - a for a, b in zip(ticks, ticks[1:]))
    assert longest > 0.3, "the queue never filled: nothing was tested"
    assert pause < longest / 2, (pause, longest)


@pytest.mark.gpu
def test_calls_from_two_threads_at_once():
    """Each thread on a stream of its own, with sizes that take both of attention's ways."""
    from unum_ops_b200 import append_cache, evict_cache, paged_attention

    cases = []
    for seed, lens in ((1, [700, 3, 90]), (2, [30000, 40, 17000])):
        q, kc, vc, table, ln = [x.to(dev()) for x in make_case(seed, lens, 2, 16, 128, 1, "bf16")]
        w = torch.rand(3, 2, table.shape[1], device=dev())
        k = torch.randn(3, 2, 128, device=dev()).to(torch.bfloat16)
        cases.append((q, kc, vc, table, ln, w, k, torch.arange(3, dtype=torch.int32, device=dev())))

    def step(q, kc, vc, table, ln, w, k, bs):
        w, kc, vc = w.clone(), kc.clone(), vc.clone()
        append_cache(k, k, kc, vc, table, bs, ln)
        out = paged_attention(q, kc, vc, table, ln, weights=w, return_lse=True)
        with pytest.raises(ValueError, match="budget"):
            evict_cache(table, ln, w, budget=0)
        return [*out, *evict_cache(table, ln, w, budget=50, init_pages=2)]

    want = [step(*c) for c in cases]
    torch.cuda.synchronize()
    got = [[], []]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(100):
                got[i].append(step(*cases[i]))
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for g, w in zip(got, want):
        assert len(g) == 100 and all(torch.equal(x, y) for r in g for x, y in zip(r, w))


FIRST_CALLS_IN_A_GRAPH = """
import sys
sys.path[:0] = [{root!r}, {tests!r}]
import torch
from test_paged_cache import make_case
from unum_ops_b200 import append_cache, evict_cache, paged_attention
for lens in ([700, 3, 90], [30000, 40, 17000]):
    q, kc, vc, table, ln = [x.cuda() for x in make_case(1, lens, 2, 16, 128, 1, "bf16")]
    w, k = torch.rand(3, 2, table.shape[1]).cuda(), torch.ones(3, 2, 128, dtype=torch.bfloat16).cuda()
    bs = torch.arange(3, dtype=torch.int32).cuda()
    start = w.clone()
    def step():
        append_cache(k, k, kc, vc, table, bs, ln)
        return [*paged_attention(q, kc, vc, table, ln, weights=w, return_lse=True), *evict_cache(table, ln, w, budget=9)]
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    g.replay()
    torch.cuda.synchronize()
    w.copy_(start)
    assert all(torch.equal(a, b) for a, b in zip(got, step()))
print("as they should be")
"""


@pytest.mark.gpu
def test_the_first_calls_of_a_process_are_captured():
    """What a first call sets up is allowed while a graph is captured."""
    code = FIRST_CALLS_IN_A_GRAPH.format(root=ROOT, tests=os.path.join(ROOT, "tests"))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "as they should be" in r.stdout, r.stderr[-2000:]
