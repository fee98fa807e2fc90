"""The paged key-value cache: append_cache, paged_attention, evict_cache.

There are no reference functions; the oracle is the operators' definition in 64 bits, computed on the
CPU from the same (rounded) inputs, position by position through the table.

Tolerances.  With eps the output type's spacing at 1, a rounding is off by eps / 2 of the value
(bf16 2^-8, fp16 2^-11).
  out: one rounding of the output (eps/2 of |out|) and one of each probability to the same type
       before the product with v (eps/2 of sum p|v| at most); sums are fp32.  So
       |err| <= eps/2 * (|out| + sum p|v|) + 2^-16 * sum p|v| for the fp32 part (the probabilities'
       exponent: |s| * log2(e) below 2^6 here, 2^-24 of it is 2^-18, plus ex2's 2^-22 and the sums).
  lse: fp32 sums of D products of fp32 magnitude |q||k| scale, 2^-20 of sum |q k| scale + 2^-18 |lse|.
  weights: fp32, relative 2^-16 of the added weight by the same exponent, plus 2^-23 of the total.
Whole numbers (tables, lengths, evicted ids) and copied rows have to be equal.
"""
import ctypes

import numpy as np
import pytest
import torch

DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------------------------------------ oracle
def tokens_of(table, b, n, page, n_tokens):
    """Token of each of the first n positions of sequence b, -1 where it is not held."""
    p = np.arange(n)
    e = table[b, p // page].astype(np.int64)
    t = e * page + p % page
    return np.where((e >= 0) & (t < n_tokens), t, -1)


def oracle_attention(q, kc, vc, table, lens, page, scale, weights=None):
    """out, lse, the weights' new values, sum p|v|, and the scores' magnitude sum |q k| * scale (largest of the row)."""
    B, Hq, D = q.shape
    n_tokens, Hk, _ = kc.shape
    G = Hq // Hk
    out, mag = np.zeros((B, Hq, D)), np.zeros((B, Hq, D))
    lse, smag = np.full((B, Hq), -np.inf), np.zeros((B, Hq))
    new = None if weights is None else weights.astype(np.float64).copy()
    add = None if weights is None else np.zeros_like(new)
    for b in range(B):
        n = int(np.clip(lens[b], 0, table.shape[1] * page))
        t = tokens_of(table, b, n, page, n_tokens)
        at = np.nonzero(t >= 0)[0]
        if not at.size:
            continue
        for g in range(Hk):
            k, v = kc[t[at], g].astype(np.float64), vc[t[at], g].astype(np.float64)
            hs = slice(g * G, g * G + G)
            qh = q[b, hs].astype(np.float64)
            s = (qh @ k.T) * scale
            m = s.max(1, keepdims=True)
            p = np.exp(s - m)
            lse[b, hs] = m[:, 0] + np.log(p.sum(1))
            p /= p.sum(1, keepdims=True)
            out[b, hs], mag[b, hs] = p @ v, p @ np.abs(v)
            smag[b, hs] = (np.abs(qh) @ np.abs(k).T).max(1) * abs(scale)
            if new is not None:
                add[b, g, at] = p.sum(0)
    if new is not None:
        new += add
    return out, lse, new, mag, smag, add


def oracle_evict(table, lens, w, budget, init, local, page):
    B, n_pages = table.shape
    new_table, gone = np.full_like(table, -1), np.full_like(table, -1)
    new_lens, new_w = np.zeros(B, np.int32), np.zeros_like(w)
    for b in range(B):
        n = int(np.clip(lens[b], 0, n_pages * page))
        used = -(-n // page)
        x = np.zeros((w.shape[1], n_pages * page))
        x[:, :n] = w[b, :, :n]
        with np.errstate(invalid="ignore"):
            score = x.reshape(w.shape[1], n_pages, page).sum((0, 2)).astype(np.float32)
        # NaN below every number; ties by the lower index
        rank = sorted(range(used), key=lambda e: (not (e < init or e >= used - local), bool(np.isnan(score[e])),
                                                  0.0 if np.isnan(score[e]) else -score[e], e))
        keep = sorted(rank[:budget]) if used > budget else list(range(used))
        out = sorted(set(range(used)) - set(keep))
        row = keep + list(range(used, n_pages))
        new_table[b, :len(row)] = table[b, row]
        gone[b, :len(out)] = table[b, out]
        new_lens[b] = n - len(out) * page
        at = [e * page + j for e in keep for j in range(page)][:new_lens[b]]
        new_w[b, :, :len(at)] = w[b][:, at]
    return new_table, new_lens, new_w, gone


# ------------------------------------------------------------------------------------------------ inputs
def make_table(rng, lens, page, width, total):
    table = np.full((len(lens), width), -1, np.int32)
    ids, off = rng.permutation(total).astype(np.int32), 0
    for b, n in enumerate(lens):
        c = -(-int(n) // page)
        table[b, :c] = ids[off:off + c]
        off += c
    return table


def make_case(seed, lens, Hk, G, D, page, dtype, spare=1):
    rng = np.random.default_rng(seed)
    width = max(-(-int(n) // page) for n in lens) + spare
    total = sum(-(-int(n) // page) for n in lens) + 3
    table = make_table(rng, lens, page, width, total)
    t = lambda *s: torch.from_numpy(rng.standard_normal(s).astype(np.float32)).to(DT[dtype])  # noqa: E731
    q, kc, vc = t(len(lens), Hk * G, D), t(total * page, Hk, D), t(total * page, Hk, D)
    return q, kc, vc, torch.from_numpy(table), torch.tensor(lens, dtype=torch.int32)


def np64(t):
    return t.detach().cpu().to(torch.float64).numpy()


def check_attention(q, kc, vc, table, lens, page, scale, out, lse, before=None, after=None):
    half = torch.finfo(q.dtype).eps / 2
    ref, rlse, rw, mag, smag, add = oracle_attention(np64(q), np64(kc), np64(vc), table.cpu().numpy(), lens.cpu().numpy(),
                                                     page, scale, None if before is None else np64(before))
    err = np.abs(np64(out) - ref)
    allow = half * (np.abs(ref) + mag) + 2.0 ** -16 * mag
    assert np.all(err <= allow), f"out off by {np.nanmax(err / np.maximum(allow, 1e-30))} of what is allowed"
    got = np64(lse)
    none = np.isneginf(rlse)
    assert np.array_equal(none, np.isneginf(got)) and not np.isnan(got).any()
    assert np.all(np.abs(got[~none] - rlse[~none]) <= (2.0 ** -20 * smag + 2.0 ** -18 * np.abs(rlse))[~none])
    if before is not None:
        w = np64(after)
        # the added weight is off by 2^-16 and by the score's own error
        rel = 2.0 ** -16 + 2.0 ** -20 * smag.max()
        assert np.all(np.abs(w - rw) <= rel * add + 2.0 ** -23 * np.abs(rw))
        assert np.array_equal(w[add == 0], np64(before)[add == 0])


def dev():
    return torch.device("cuda", 0)


def run_attention(q, kc, vc, table, lens, page=1, weights=None, scale=None, **kw):
    import unum_ops_b200

    d = dev()
    w = None if weights is None else weights.to(d)
    out, lse = unum_ops_b200.paged_attention(q.to(d), kc.to(d), vc.to(d), table.to(d), lens.to(d), page_size=page, weights=w,
                                             return_lse=True, softmax_scale=scale, **kw)
    torch.cuda.synchronize()
    return out, lse, w


# ------------------------------------------------------------------------------------------------ refusals (CPU)
@pytest.fixture(scope="module")
def lib():
    import unum_ops_b200

    unum_ops_b200.build()
    return unum_ops_b200.load()


def attend_args(**over):
    a = dict(q=1024, B=2, Hq=32, D=128, q_sb=4096, q_sh=128, kc=2048, vc=4096, dtype=1, n_tokens=64, Hk=2, k_st=256, k_sh=128,
             v_st=256, v_sh=128, table=4096, n_pages=4, bt=4, page=16, lens=4096, max_len=64, scale=0.1, out=8192, lse=None,
             w=None, w_sb=0, w_sh=0, ws=4096, nbytes=1 << 30, stream=None)
    a.update(over)
    a["scale"] = ctypes.c_float(a["scale"])
    return list(a.values())


@pytest.mark.parametrize("over,rc,word", [
    (dict(dtype=0), -1, b"dtype"), (dict(Hq=33), -1, b"multiple"), (dict(D=96), -2, b"head_dim"),
    (dict(Hq=130, Hk=2), -2, b"heads"), (dict(page=24), -1, b"page_size"), (dict(page=0), -1, b"page_size"),
    (dict(q=0), -1, b"null"), (dict(lens=0), -1, b"null"), (dict(table=0), -1, b"null"), (dict(kc=2056), -1, b"aligned"),
    (dict(k_st=252), -1, b"multiples"), (dict(q_sh=4), -1, b"multiples"), (dict(max_len=65), -1, b"max_seqlen"),
    (dict(B=-1), -1, b"sizes"), (dict(ws=0), -4, b"workspace"), (dict(nbytes=0), -4, b"workspace"), (dict(B=0), 0, b"")])
def test_attention_entry_refuses(lib, over, rc, word):
    assert lib.unum_paged_attention(*attend_args(**over)) == rc
    assert word in lib.unum_last_error()


@pytest.mark.parametrize("over,rc", [(dict(D=80), -2), (dict(page=3), -1), (dict(k=8), -1), (dict(kc_st=100), -1), (dict(bs=0), -1),
                                     (dict(T=0), 0), (dict(n_pages=0), 0), (dict(T=-1), -1)])
def test_append_entry_refuses(lib, over, rc):
    a = dict(k=1024, v=1024, T=4, Hk=2, D=128, k_st=256, k_sh=128, v_st=256, v_sh=128, kc=2048, vc=4096, n_tokens=64, kc_st=256,
             kc_sh=128, vc_st=256, vc_sh=128, table=1024, B=2, n_pages=4, bt=4, page=16, bs=1024, pos=1024, stream=None)
    a.update(over)
    assert lib.unum_cache_append(*a.values()) == rc


@pytest.mark.parametrize("over,rc", [(dict(page=6), -1), (dict(local=0), -1), (dict(init=-1), -1), (dict(budget=4), -1),
                                     (dict(n_pages=409601), -2), (dict(n_pages=1 << 16, page=1 << 15), -1), (dict(w=0), -1),
                                     (dict(lens=0), -1), (dict(B=0), 0), (dict(Hk=0), -1)])
def test_evict_entry_refuses(lib, over, rc):
    a = dict(table=1024, B=2, n_pages=16, bt=16, lens=1024, w=1024, Hk=2, w_sb=512, w_sh=256, page=16, budget=5, init=2, local=3,
             nt=1024, nl=1024, nw=1024, gone=1024, stream=None)
    a.update(over)
    assert lib.unum_cache_evict(*a.values()) == rc


def test_cpu_tensors_are_refused(lib):
    from unum_ops_b200 import append_cache, evict_cache, paged_attention

    q, kc, vc, table, lens = make_case(1, [5, 9], 2, 4, 64, 1, "bf16")
    with pytest.raises(ValueError, match="CUDA"):
        paged_attention(q, kc, vc, table, lens)
    with pytest.raises(ValueError, match="CUDA"):
        append_cache(kc[:2].clone(), vc[:2].clone(), kc, vc, table, lens, lens)
    with pytest.raises(ValueError, match="CUDA"):
        evict_cache(table, lens, torch.zeros(2, 2, table.shape[1]), budget=4)


def test_attention_wrapper_refuses(lib):
    from unum_ops_b200 import paged_attention

    q, kc, vc, table, lens = make_case(1, [5, 9], 2, 4, 64, 1, "bf16")
    W = table.shape[1]
    bad = [
        (dict(q=q.float()), ValueError), (dict(q=q[:, :7]), ValueError), (dict(q=q[..., :32]), ValueError),
        (dict(kc=kc.float(), vc=vc.float()), ValueError), (dict(vc=vc[:-1]), ValueError), (dict(vc=vc.half()), ValueError),
        (dict(kc=kc[..., ::2], vc=vc[..., ::2], q=q[..., ::2]), ValueError),
        (dict(table=table[:1]), ValueError), (dict(lens=lens[:1]), ValueError), (dict(page_size=3), ValueError),
        (dict(page_size=0), ValueError), (dict(max_seqlen=-1), ValueError),
        (dict(weights=torch.zeros(2, 2, W - 1)), ValueError), (dict(weights=torch.zeros(2, 1, W)), ValueError),
        (dict(weights=torch.zeros(2, 2, W, dtype=torch.float64)), ValueError),
        (dict(weights=torch.zeros(1, 2, W).expand(2, 2, W)), ValueError),
        (dict(weights=torch.zeros(2, 2, 2 * W)[..., ::2]), ValueError),
        (dict(q=q.clone().requires_grad_()), NotImplementedError), (dict(kc=kc.clone().requires_grad_()), NotImplementedError),
        (dict(weights=torch.zeros(2, 2, W, requires_grad=True)), NotImplementedError),
    ]
    for over, error in bad:
        a = dict(q=q, kc=kc, vc=vc, table=table, lens=lens)
        a.update(over)
        with pytest.raises(error):
            paged_attention(a.pop("q"), a.pop("kc"), a.pop("vc"), a.pop("table"), a.pop("lens"), **a)


def test_append_and_evict_wrappers_refuse(lib):
    from unum_ops_b200 import append_cache, evict_cache

    _, kc, vc, table, lens = make_case(1, [5, 9], 2, 4, 64, 1, "bf16")
    k, i = kc[:2].clone(), torch.zeros(2, dtype=torch.int32)
    for a in [(kc[3:5], k, kc, vc), (k, vc[-2:], kc, vc)]:
        with pytest.raises(ValueError, match="memory"):
            append_cache(*a, table, i, i)
    with pytest.raises(TypeError):
        append_cache(k, [1], kc, vc, table, i, i)
    with pytest.raises(TypeError):
        append_cache(k, k, kc, vc, table, i, i, page_size=1.5)
    for a in [(k.float(), k, kc, vc), (k[:, :1], k[:, :1], kc, vc), (k, k[:1], kc, vc), (k, k, kc, kc),
              (k, k, kc[:1].expand(12, 2, 64), vc[:12]), (k, k, kc[:, :1].expand(-1, 2, -1), vc)]:
        with pytest.raises(ValueError):
            append_cache(*a, table, i, i)
    with pytest.raises(ValueError):
        append_cache(k, k, kc, vc, table, i[:1], i)
    with pytest.raises(NotImplementedError):
        append_cache(k.clone().requires_grad_(), k, kc, vc, table, i, i)
    w = torch.zeros(2, 2, table.shape[1])
    for kw in [dict(budget=0), dict(budget=3, local_pages=4), dict(budget=3, local_pages=0), dict(budget=3, init_pages=-1),
               dict(budget=3, init_pages=3), dict(budget=3, page_size=5), dict(budget=3, page_size=2)]:
        with pytest.raises(ValueError):
            evict_cache(table, lens, w, **kw)
    with pytest.raises(ValueError):
        evict_cache(table, lens, w.double(), budget=3)
    with pytest.raises(ValueError):
        evict_cache(table, lens[:1], w, budget=3)


# ------------------------------------------------------------------------------------------------ attention (GPU)
ATTEND = [
    # lens, Hk, G, D, page, dtype
    ([1], 1, 1, 64, 1, "bf16"), ([1, 0, 2], 2, 16, 128, 1, "bf16"), ([0], 2, 16, 128, 1, "bf16"),
    ([15, 16, 17, 31, 33, 63, 64, 65], 2, 16, 128, 1, "bf16"), ([127, 128, 129, 255, 257], 1, 8, 128, 16, "fp16"),
    ([1000], 2, 16, 128, 1, "bf16"), ([700, 3, 0, 411], 8, 4, 64, 16, "fp16"), ([333, 90], 2, 32, 128, 64, "bf16"),
    ([513, 1], 1, 64, 128, 2, "bf16"), ([260, 77], 2, 33, 64, 128, "fp16"), ([97, 200], 3, 5, 128, 4, "bf16"),
    ([5000], 1, 16, 128, 1, "bf16"), ([2111, 4096, 1], 2, 16, 64, 32, "bf16"), ([50] * 40, 2, 17, 128, 1, "fp16"),
    ([130, 20, 64], 4, 1, 128, 256, "bf16"), ([9000, 1, 0, 300], 2, 16, 128, 1, "fp16"), ([64] * 3, 1, 48, 64, 64, "bf16"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("lens,Hk,G,D,page,dtype", ATTEND)
@pytest.mark.parametrize("gather", [False, True])
def test_attention(lens, Hk, G, D, page, dtype, gather):
    q, kc, vc, table, ln = make_case(len(lens) * 1000 + max(lens) + G, lens, Hk, G, D, page, dtype)
    before = None
    if gather:
        before = torch.from_numpy(np.random.default_rng(5).random((len(lens), Hk, table.shape[1] * page)).astype(np.float32))
    out, lse, after = run_attention(q, kc, vc, table, ln, page, before)
    check_attention(q, kc, vc, table, ln, page, D ** -0.5, out, lse, before, after)


# Work that is dealt out in units and joined by the second kernel: more than the clusters take.
DEALT = [
    ([20000], 2, 16, 128, 1, "bf16"), ([40000, 5, 0, 1300], 1, 8, 64, 16, "fp16"), ([1500, 3, 0, 2000] + [700] * 40, 2, 32, 128, 64, "bf16"),
    ([17000, 4000], 2, 64, 128, 2, "bf16"), ([33000, 1], 1, 33, 64, 128, "fp16"), ([100] * 200, 2, 5, 128, 4, "bf16"),
    ([0] * 150 + [65, 0, 64, 1, 0, 129, 3000], 2, 16, 128, 1, "fp16"), ([70000], 1, 1, 64, 1, "bf16"), ([12345] * 3, 4, 20, 64, 32, "bf16"),
    (list(range(0, 900, 3)), 1, 16, 128, 16, "bf16"), ([31, 33] * 80, 1, 40, 128, 8, "fp16"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("lens,Hk,G,D,page,dtype", DEALT)
@pytest.mark.parametrize("gather", [False, True])
def test_attention_dealt_out(lens, Hk, G, D, page, dtype, gather):
    test_attention(lens, Hk, G, D, page, dtype, gather)


@pytest.mark.gpu
@pytest.mark.parametrize("bound", [1000, 1024, 1025, 5000, 16384, 16385, 30000])
def test_attention_the_bound_of_the_lengths_changes_the_split_only(bound):
    """The same sequences under several host-side bounds (each another split of the work), all within tolerance."""
    lens = [1000, 999, 0, 513]
    q, kc, vc, table, ln = make_case(31, lens, 2, 16, 128, 1, "bf16", spare=bound - 1000)
    before = torch.rand(4, 2, table.shape[1], generator=torch.Generator().manual_seed(2))
    out, lse, after = run_attention(q, kc, vc, table, ln, 1, before, max_seqlen=bound)
    check_attention(q, kc, vc, table, ln, 1, 128 ** -0.5, out, lse, before, after)


@pytest.mark.gpu
@pytest.mark.parametrize("B", [2, 200])
def test_attention_over_nothing(B):
    """A table without a page, a cache without a token, a batch without a sequence."""
    from unum_ops_b200 import paged_attention

    d = dev()
    q, kc = torch.randn(B, 32, 128, device=d, dtype=torch.bfloat16), torch.randn(9, 2, 128, device=d, dtype=torch.bfloat16)
    i32 = dict(dtype=torch.int32, device=d)
    for k, table in ((kc, torch.zeros(B, 0, **i32)), (kc[:0], torch.zeros(B, 7, **i32))):
        w = torch.ones(B, 2, 7, device=d)
        out, lse = paged_attention(q, k, k, table, torch.full((B,), 5, **i32), weights=w, return_lse=True)
        assert not out.any() and torch.isneginf(lse).all() and (w == 1).all()
    out = paged_attention(q[:0], kc, kc, torch.zeros(0, 3, **i32), torch.zeros(0, **i32))
    assert out.shape == (0, 32, 128)


@pytest.mark.gpu
def test_attention_positions_that_are_not_held():
    """Table entries outside the cache (negative, past its end, a page that its end cuts) hide their positions; what a
    hidden or unused row of the cache holds (NaN, infinities) does not matter."""
    page = 8
    q, kc, vc, table, ln = make_case(3, [100, 64, 40, 17], 2, 16, 128, page, "bf16")
    n_tokens = kc.shape[0] - 3  # the last page is cut
    cut = kc.shape[0] // page - 1
    table[0, 2], table[0, 5], table[1, 0], table[1, 3] = -1, 1 << 28, cut, -(1 << 30)
    table[2, :] = -5  # a row that leaves nothing
    table[3, 2] = (1 << 31) - 1
    used = set()
    for b, n in enumerate(ln.tolist()):
        used |= set(tokens_of(table.numpy(), b, n, page, n_tokens).tolist())
    unused = [t for t in range(kc.shape[0]) if t not in used]
    kc[unused], vc[unused] = float("nan"), float("inf")
    kc, vc = kc[:n_tokens], vc[:n_tokens]
    before = torch.rand(4, 2, table.shape[1] * page, generator=torch.Generator().manual_seed(1))
    out, lse, after = run_attention(q, kc, vc, table, ln, page, before)
    assert torch.isneginf(lse[2]).all() and not out[2].any()
    check_attention(q, kc, vc, table, ln, page, 128 ** -0.5, out, lse, before, after)


@pytest.mark.gpu
def test_attention_values_at_the_border():
    """Lowest and largest values, infinities and NaN in rows that are attended to."""
    lens = [300, 300, 300, 200]
    q, kc, vc, table, ln = make_case(4, lens, 1, 4, 64, 1, "bf16")
    t = table.numpy()
    big = torch.finfo(torch.bfloat16).max
    kc[t[0, 7]] = float("nan")          # all scores of that position: every output is NaN
    vc[t[1, 9], :, 5] = float("inf")    # one dim of the values
    q[2] = 0                            # equal scores
    q[3, :, :] = 0
    q[3, :, 0] = 1
    kc[t[3, :200], 0, 0] = -big         # scores near the type's lowest value
    kc[t[3, 50], 0, 0] = -big / 2
    out, lse, _ = run_attention(q, kc, vc, table, ln)
    assert torch.isnan(out[0]).all() and torch.isnan(lse[0]).all()
    assert torch.isinf(out[1, :, 5]).all() and torch.isfinite(out[1, :, :5]).all() and torch.isfinite(out[1, :, 6:]).all()
    c = lambda x: x[2:]  # noqa: E731
    ref, rlse, _, mag, _, _ = oracle_attention(np64(c(q)), np64(kc), np64(vc), t[2:], lens[2:], 1, 64 ** -0.5)
    assert np.all(np.abs(np64(out[2:]) - ref) <= 2.0 ** -8 * (np.abs(ref) + mag) + 2.0 ** -16 * mag)
    np.testing.assert_allclose(np64(lse[2:]), rlse, rtol=2.0 ** -18)
    # scores that are all -inf count as none
    kc[t[3, :200], 0, 0] = float("-inf")
    out, lse, _ = run_attention(q, kc, vc, table, ln)
    assert torch.isneginf(lse[3]).all() and not out[3].any()


@pytest.mark.gpu
def test_attention_scale_strides_and_lengths_out_of_range():
    """A negative scale, q and the caches as views of larger tensors, lengths that are clamped, int64 tables."""
    import unum_ops_b200

    d = dev()
    lens = [70, 333]
    q, kc, vc, table, ln = make_case(6, lens, 2, 16, 128, 1, "bf16")
    n = kc.shape[0]
    kv = torch.zeros(n, 2, 3, 128, dtype=torch.bfloat16)
    kv[:, 0, 1:], kv[:, 1, 1:] = kc, vc
    kv = kv.to(d)
    qq = torch.zeros(2, 40, 128, dtype=torch.bfloat16, device=d)
    qq[:, 4:36] = q.to(d)
    out, lse = unum_ops_b200.paged_attention(qq[:, 4:36], kv[:, 0, 1:], kv[:, 1, 1:], table.to(d).long(), ln.to(d).long(),
                                             softmax_scale=-0.25, return_lse=True)
    check_attention(q, kc, vc, table, ln, 1, -0.25, out, lse)
    # a q that 16-byte loads cannot read
    odd = torch.zeros(2, 32, 129, dtype=torch.bfloat16, device=d)
    odd[..., 1:] = q.to(d)
    again = unum_ops_b200.paged_attention(odd[..., 1:], kv[:, 0, 1:], kv[:, 1, 1:], table.to(d), ln.to(d), softmax_scale=-0.25)
    assert torch.equal(again, out)
    # lengths outside [0, max_seqlen]
    far = torch.tensor([-7, 1 << 30], dtype=torch.int32)
    out, lse, _ = run_attention(q, kc, vc, table, far, max_seqlen=333)
    check_attention(q, kc, vc, table, torch.tensor([0, 333]), 1, 128 ** -0.5, out, lse)
    out, lse, _ = run_attention(q, kc, vc, table, ln, max_seqlen=100)
    check_attention(q, kc, vc, table, torch.tensor([70, 100]), 1, 128 ** -0.5, out, lse)


@pytest.mark.gpu
def test_attention_offsets_past_32_bits():
    """A cache of more than 2^31 elements: rows at both of its ends."""
    n, d = (1 << 23) + 5000, dev()   # 8.4 M tokens x 2 heads x 128: 2^31 elements and more, 4.3 GB a tensor
    kc, vc = (torch.empty(n, 2, 128, dtype=torch.bfloat16, device=d) for _ in range(2))
    rng = np.random.default_rng(9)
    rows = np.concatenate([rng.permutation(4000)[:500], n - 1 - rng.permutation(4000)[:500]])
    rng.shuffle(rows)
    at = torch.from_numpy(rows).to(d)
    k, v = (torch.from_numpy(rng.standard_normal((1000, 2, 128)).astype(np.float32)).to(torch.bfloat16) for _ in range(2))
    kc[at], vc[at] = k.to(d), v.to(d)
    q = torch.from_numpy(rng.standard_normal((1, 32, 128)).astype(np.float32)).to(torch.bfloat16)
    table = torch.from_numpy(rows.astype(np.int32))[None]
    ln = torch.tensor([1000])
    out, lse, _ = run_attention(q, kc, vc, table, ln)
    check_attention(q, k, v, torch.arange(1000, dtype=torch.int32)[None], ln, 1, 128 ** -0.5, out, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[3000, 40, 0, 1777], [30000, 40, 0, 17771]])
def test_attention_same_bits_again_and_in_a_graph(lens):
    """Two calls give the same bits; a captured call follows its inputs; two graphs replayed on two streams at once do not
    share a workspace."""
    import unum_ops_b200

    d = dev()
    q, kc, vc, table, ln = [x.to(d) for x in make_case(12, lens, 2, 16, 128, 1, "bf16")]
    w = torch.zeros(4, 2, table.shape[1], device=d)
    call = lambda: unum_ops_b200.paged_attention(q, kc, vc, table, ln, weights=w, return_lse=True)  # noqa: E731
    a, la = call()
    wa = w.clone()
    w.zero_()
    b, lb = call()
    assert torch.equal(a, b) and torch.equal(la, lb) and torch.equal(wa, w)
    w2 = torch.zeros_like(w)
    graphs = []
    for weights in (w, w2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = unum_ops_b200.paged_attention(q, kc, vc, table, ln, weights=weights, return_lse=True)
        graphs.append((g, o))
    ln.copy_(torch.tensor([2999, 41, 7, 100], dtype=torch.int32))
    q.mul_(0.5)
    w.zero_()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        for (g, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    fresh = torch.zeros_like(w)
    want, wl = unum_ops_b200.paged_attention(q, kc, vc, table, ln, weights=fresh, return_lse=True)
    for _ in range(4):
        unum_ops_b200.paged_attention(q, kc, vc, table, ln, weights=fresh)
    for (g, (o, l)), weights in zip(graphs, (w, w2)):
        assert torch.equal(o, want) and torch.equal(l, wl) and torch.equal(weights, fresh)


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[500, 40, 0, 177], [30000, 40, 0, 17771]])
def test_calls_behind_kernels_that_still_run(lens):
    """Kernels are launched while the one before them runs: what that one writes (q, the cache, the lengths, the table)
    is waited for, and so is what the calls themselves leave for the next kernel.  No synchronisation inside."""
    from unum_ops_b200 import append_cache, evict_cache, paged_attention

    d = dev()
    q, kc, vc, table, ln = [x.to(d) for x in make_case(14, lens, 2, 16, 128, 1, "bf16")]
    W = table.shape[1]
    slow = torch.randn(3000, 3000, device=d)
    want = paged_attention(q, kc, vc, table, ln, return_lse=True)
    w = torch.rand(4, 2, W, device=d)
    want_evicted = evict_cache(table, ln, w, budget=100)
    k, v = torch.randn(2, 300, 2, 128, device=d, dtype=torch.bfloat16)
    rows = torch.arange(300, device=d, dtype=torch.int32)
    torch.cuda.synchronize()
    for _ in range(4):
        q2, k2, t2, l2, w2 = torch.zeros_like(q), torch.zeros_like(kc), torch.zeros_like(table), torch.zeros_like(ln), torch.zeros_like(w)
        vc2, got = torch.full_like(vc, 9), []
        torch.mm(slow, slow)
        t2.copy_(table)
        l2.copy_(ln)
        w2.copy_(w)
        q2.copy_(q)
        vc2.copy_(vc)
        k2.copy_(kc)  # the last and the largest: still running when the call is made
        got.append(paged_attention(q2, k2, vc2, t2, l2, return_lse=True))
        w2.mul_(1.0)
        got.append(evict_cache(t2, l2, w2, budget=100))
        first, n = got[1][0], got[1][1]
        got.append(paged_attention(q2, k2, vc2, first, n, return_lse=True))
        append_cache(k, v, k2, vc2, rows[None].expand(1, -1), torch.zeros_like(rows), rows + 1)
        got.append((k2[:300].clone(), vc2[:300].clone()))
        got.append(paged_attention(q2, k2, vc2, t2, l2, return_lse=True))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got[0], want))
        assert all(torch.equal(a, b) for a, b in zip(got[1], want_evicted))
        shorter = paged_attention(q, kc, vc, want_evicted[0], want_evicted[1], return_lse=True)
        assert all(torch.equal(a, b) for a, b in zip(got[2], shorter))
        assert torch.equal(got[3][0], k) and torch.equal(got[3][1], v)
        kc3, vc3 = kc.clone(), vc.clone()
        kc3[:300], vc3[:300] = k, v
        assert all(torch.equal(a, b) for a, b in zip(got[4], paged_attention(q, kc3, vc3, table, ln, return_lse=True)))


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[900, 20, 300], [30000, 20, 17000]])
def test_calls_on_several_streams_at_once(lens):
    """Calls that overlap have workspaces of their own."""
    from unum_ops_b200 import paged_attention

    q, kc, vc, table, ln = [x.to(dev()) for x in make_case(3, lens, 2, 16, 128, 1, "bf16")]
    qs = [q * (i + 1) / 3 for i in range(4)]
    want = [paged_attention(x, kc, vc, table, ln, return_lse=True) for x in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    for _ in range(20):
        got = []
        for s, x in zip(streams, qs):
            with torch.cuda.stream(s):
                got.append(paged_attention(x, kc, vc, table, ln, return_lse=True))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))


@pytest.mark.gpu
def test_large_batches():
    """More sequences than there are threads in a block, or blocks on the GPU."""
    from unum_ops_b200 import evict_cache

    rng = np.random.default_rng(8)
    for B, longest, Hk, G in ((6000, 40, 1, 4), (1500, 300, 2, 16), (70000, 3, 1, 1)):
        lens = rng.integers(0, longest + 1, B)
        q, kc, vc, table, _ = make_case(7, np.maximum(lens, 1), Hk, G, 64, 1, "bf16")
        ln = torch.from_numpy(lens.astype(np.int32))
        before = torch.from_numpy(rng.random((B, Hk, table.shape[1])).astype(np.float32))
        out, lse, after = run_attention(q, kc, vc, table, ln, 1, before)
        check_attention(q, kc, vc, table, ln, 1, 64 ** -0.5, out, lse, before, after)
    lens, w = rng.integers(0, 201, 2000).astype(np.int32), rng.random((2000, 2, 200)).astype(np.float32)
    table = np.arange(2000 * 200, dtype=np.int32).reshape(2000, 200)
    got = evict_cache(*[torch.from_numpy(x).to(dev()) for x in (table, lens, w)], budget=64, local_pages=3)
    for x, y in zip(got, oracle_evict(table, lens, w, 64, 0, 3, 1)):
        np.testing.assert_array_equal(x.cpu().numpy(), y)


# ------------------------------------------------------------------------------------------------ append (GPU)
@pytest.mark.gpu
@pytest.mark.parametrize("T,B,Hk,D,page,dtype", [(1, 1, 2, 128, 1, "bf16"), (7, 3, 1, 64, 4, "fp16"), (500, 5, 8, 64, 16, "bf16"),
                                                 (333, 2, 3, 128, 64, "fp16"), (2500, 1, 2, 128, 1, "bf16")])
def test_append(T, B, Hk, D, page, dtype):
    from unum_ops_b200 import append_cache

    rng = np.random.default_rng(T)
    d = dev()
    new = rng.multinomial(T, [1 / B] * B)
    had = rng.integers(0, 40, B)
    lens = new + had
    total = sum(-(-int(n) // page) for n in lens) + 3
    table = make_table(rng, lens, page, max(-(-int(n) // page) for n in lens) + 1, total)
    bs = np.repeat(np.arange(B), new).astype(np.int32)
    pos = np.concatenate([h + 1 + np.arange(n) for h, n in zip(had, new)]).astype(np.int32)
    # some that are not to be written
    if T > 6:
        bs[1], bs[2], pos[3], pos[4] = -1, B, 0, table.shape[1] * page + 1
        e = pos[5] - 1
        table[bs[5], e // page] = total * 2
    kv = torch.from_numpy(rng.standard_normal((T, 3 * Hk, D)).astype(np.float32)).to(DT[dtype])
    cache = torch.from_numpy(rng.standard_normal((total * page, 2, Hk, D)).astype(np.float32)).to(DT[dtype])
    want, p = cache.clone(), pos.astype(np.int64) - 1
    for t in range(T):
        if 0 <= bs[t] < B and 0 <= p[t] < table.shape[1] * page:
            e = int(table[bs[t], p[t] // page])
            if 0 <= e < total:
                want[e * page + p[t] % page, 0], want[e * page + p[t] % page, 1] = kv[t, Hk:2 * Hk], kv[t, 2 * Hk:]
    gkv, g = kv.to(d), cache.to(d)
    got = append_cache(gkv[:, Hk:2 * Hk], gkv[:, 2 * Hk:], g[:, 0], g[:, 1], torch.from_numpy(table).to(d),
                       torch.from_numpy(bs).to(d), torch.from_numpy(pos).to(d), page_size=page)
    assert got[0].data_ptr() == g.data_ptr()
    assert torch.equal(g.cpu(), want)


@pytest.mark.gpu
def test_append_rows_that_wide_loads_cannot_read():
    from unum_ops_b200 import append_cache

    d = dev()
    kv = torch.randn(5, 2, 65, device=d, dtype=torch.bfloat16)[..., 1:]
    kc, vc = torch.zeros(2, 8, 2, 64, device=d, dtype=torch.bfloat16)
    table = torch.arange(8, device=d, dtype=torch.int32)[None].flip(1)
    append_cache(kv, kv, kc, vc, table, torch.zeros(5, device=d), torch.arange(1, 6, device=d))
    assert torch.equal(kc[3:].flip(0), kv) and torch.equal(vc[3:].flip(0), kv) and not kc[:3].any()
    append_cache(kv[:0], kv[:0], kc, vc, table, torch.zeros(0, device=d), torch.zeros(0, device=d))


# ------------------------------------------------------------------------------------------------ evict (GPU)
EVICT = [
    # lens, Hk, page, budget, init, local, kind of weights
    ([5], 1, 1, 3, 0, 1, "random"), ([1, 0, 2, 3], 2, 1, 2, 1, 1, "random"), ([100, 64, 65, 7], 2, 1, 64, 4, 16, "random"),
    ([1000, 999], 2, 1, 300, 0, 1, "ties"), ([1000, 40], 3, 16, 20, 1, 2, "random"), ([513, 77], 1, 2, 100, 0, 7, "ties"),
    ([4000, 4096, 1], 2, 64, 9, 1, 2, "random"), ([300], 2, 1, 10, 4, 6, "random"), ([20000, 3], 2, 1, 5000, 10, 100, "random"),
    ([2048], 2, 1, 1024, 0, 1, "equal"), ([700], 2, 4, 50, 2, 2, "odd"), ([150000], 1, 1, 70000, 5, 9, "random"),
    ([9000], 2, 256, 7, 0, 1, "negative"), ([50] * 30, 2, 8, 3, 1, 1, "ties"),
    ([409598], 1, 1, 300001, 3, 1, "random"), ([120000, 90000, 5], 2, 1, 60000, 3, 1, "ties"), ([33] * 5, 4, 32, 1, 0, 1, "random"),
]


def make_weights(rng, kind, shape):
    w = np.exp(2 * rng.standard_normal(shape)).astype(np.float32)
    if kind == "ties":
        w = rng.integers(0, 4, shape).astype(np.float32)
    if kind == "equal":
        w[:] = 0.25
    if kind == "negative":
        w = rng.standard_normal(shape).astype(np.float32)
    if kind == "odd":
        w[..., rng.integers(0, shape[-1], 40)] = np.nan
        w[..., rng.integers(0, shape[-1], 40)] = np.inf
        w[..., rng.integers(0, shape[-1], 40)] = -np.inf
        w[..., rng.integers(0, shape[-1], 40)] = -0.0
    return w


@pytest.mark.gpu
@pytest.mark.parametrize("lens,Hk,page,budget,init,local,kind", EVICT)
def test_evict(lens, Hk, page, budget, init, local, kind):
    from unum_ops_b200 import evict_cache

    rng = np.random.default_rng(len(lens) + lens[0] + page)
    width = max(-(-n // page) for n in lens) + 2
    table = rng.permutation(len(lens) * width).reshape(len(lens), width).astype(np.int32)  # pages behind the lengths too
    w = make_weights(rng, kind, (len(lens), Hk, width * page))
    d = dev()
    ln = np.array(lens, np.int32)
    args = [torch.from_numpy(x).to(d) for x in (table, ln, w)]
    got = evict_cache(*args, budget=budget, init_pages=init, local_pages=local, page_size=page)
    want = oracle_evict(table, ln, w, budget, init, local, page)
    for name, x, y in zip(("table", "seqlens", "weights", "evicted"), got, want):
        np.testing.assert_array_equal(x.cpu().numpy(), y, err_msg=name)
    for x, y in zip(args, (table, ln, w)):
        np.testing.assert_array_equal(x.cpu().numpy(), y)  # the inputs stay


@pytest.mark.gpu
def test_evict_strides_and_lengths_out_of_range():
    from unum_ops_b200 import evict_cache

    rng = np.random.default_rng(2)
    d = dev()
    table = rng.permutation(3 * 40).reshape(3, 40).astype(np.int32)
    w = rng.random((2, 3, 7 + 80)).astype(np.float32)
    ln = np.array([-3, 1 << 30, 33], np.int32)
    big = torch.from_numpy(np.concatenate([table, table], 1)).to(d).long()
    got = evict_cache(big[:, :40], torch.from_numpy(ln).to(d), torch.from_numpy(w).to(d).transpose(0, 1)[..., 7:], budget=6,
                      init_pages=1, local_pages=2, page_size=2)
    want = oracle_evict(table, ln, w.transpose(1, 0, 2)[..., 7:], 6, 1, 2, 2)
    for x, y in zip(got, want):
        np.testing.assert_array_equal(x.cpu().numpy(), y)


# ------------------------------------------------------------------------------------------------ together (GPU)
@pytest.mark.gpu
def test_a_decode_loop_with_eviction():
    """A prompt is written, then tokens one by one: write, attend, gather, and every few steps shorten; each step is
    checked against a cache kept in plain lists."""
    from unum_ops_b200 import append_cache, evict_cache, paged_attention

    rng = np.random.default_rng(77)
    d = dev()
    page, B, Hk, G, D, budget = 4, 3, 2, 16, 128, 12
    n_pages, total = 40, 90
    free = [int(x) for x in rng.permutation(total)]
    kc, vc = (torch.zeros(total * page, Hk, D, dtype=torch.bfloat16, device=d) for _ in range(2))
    table = torch.full((B, n_pages), -1, dtype=torch.int32, device=d)
    weights = torch.zeros(B, Hk, n_pages * page, device=d)
    held = [[] for _ in range(B)]        # (key, value) of each position
    wref = [[] for _ in range(B)]        # [Hk] gathered, in 64 bits

    def rows(*shape):
        return torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).to(torch.bfloat16)

    def write(counts):
        bs, pos = [], []
        for b, n in enumerate(counts):
            for _ in range(n):
                at = len(held[b])
                if at % page == 0:
                    table[b, at // page] = free.pop()
                k, v = rows(Hk, D), rows(Hk, D)
                held[b].append((k, v))
                wref[b].append(np.zeros(Hk))
                bs.append(b)
                pos.append(at + 1)
        k, v = (torch.stack([held[b][p - 1][i] for b, p in zip(bs, pos)]).to(d) for i in (0, 1))
        append_cache(k, v, kc, vc, table, torch.tensor(bs, device=d), torch.tensor(pos, device=d), page_size=page)

    write([30, 7, 70])
    for step in range(24):
        write([1, 1, 1])
        lens = torch.tensor([len(x) for x in held], dtype=torch.int32, device=d)
        q = rows(B, Hk * G, D)
        before = weights.clone()
        out, lse = paged_attention(q.to(d), kc, vc, table, lens, page_size=page, weights=weights, return_lse=True)
        check_attention(q, kc, vc, table, lens, page, D ** -0.5, out, lse, before, weights)
        for b in range(B):
            k, v = (np.stack([np64(x[i]) for x in held[b]]) for i in (0, 1))
            o, _, add, mag, _, _ = oracle_attention(np64(q[b:b + 1]), k, v, np.arange(len(k), dtype=np.int32)[None], [len(k)], 1,
                                                    D ** -0.5, np.zeros((1, Hk, len(k))))
            assert np.all(np.abs(np64(out[b]) - o[0]) <= 2.0 ** -8 * (np.abs(o[0]) + mag[0]) + 2.0 ** -16 * mag[0])
            for p in range(len(k)):
                wref[b][p] = wref[b][p] + add[0, :, p]
            np.testing.assert_allclose(np64(weights[b, :, :len(k)]), np.stack(wref[b], 1), rtol=1e-4)
        if step % 6 == 5:
            table, lens, weights, gone = evict_cache(table, lens, weights, budget=budget, init_pages=1, local_pages=2,
                                                     page_size=page)
            for b in range(B):
                used = -(-len(held[b]) // page)
                sums = [sum(wref[b][p].sum() for p in range(e * page, min(len(held[b]), e * page + page))) for e in range(used)]
                rank = sorted(range(used), key=lambda e: (not (e < 1 or e >= used - 2), -sums[e], e))
                keep = sorted(rank[:budget])
                held[b] = [held[b][p] for e in keep for p in range(e * page, min(len(held[b]), e * page + page))]
                wref[b] = [wref[b][p] for e in keep for p in range(e * page, min(len(wref[b]), e * page + page))]
                freed = [x for x in gone[b].tolist() if x >= 0]
                assert len(freed) == used - len(keep) and int(lens[b]) == len(held[b])
                free += freed


@pytest.mark.gpu
def test_the_same_cache_serves_sparse_attention():
    """With page size 1, sparse_attention over every block of a short sequence is paged_attention over its cache."""
    from unum_ops_b200 import paged_attention, sparse_attention

    d = dev()
    lens = [640, 129, 1]
    q, kc, vc, table, ln = [x.to(d) for x in make_case(21, lens, 2, 16, 128, 1, "bf16")]
    K = 10
    topk = torch.arange(K, device=d, dtype=torch.int32).expand(2, 3, K).contiguous()
    tb = torch.arange(3, device=d, dtype=torch.int32)
    a = sparse_attention(q, kc, vc, topk, table, tb, ln, ln, head_group=2)
    b = paged_attention(q, kc, vc, table, ln)
    # both round the probabilities and the output to bf16 once
    mag = float(vc.float().abs().max())
    assert (a.float() - b.float()).abs().max() <= 4 * 2.0 ** -8 * mag
