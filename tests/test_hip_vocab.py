"""Losses over a large vocabulary (gridmm_amd/vocab.py, csrc/vocab_loss.hip) and the selection of top logits (csrc/top_logits.hip)
against their definitions in 64 bits.

Tolerances are bounds, derived from the arithmetic (u = 2^-24 is half a step of fp32):
  score      two fp16 planes hold 22 bits of an fp32 operand and the lo lo product is left out: 3 2^-22 of |h| |W|; 16-bit products
             are exact; an fp32 sum of n terms is off by n u of the sum of their sizes; three roundings and a base-2 scale on |z|
             e_z = (c + K u) |h| . |W| + 4 u |z|,   c = 3 2^-22 (fp32), 0 (16 bits)
  loss       L is off by at most max e_z + the sum of exponentials (V u + 2 steps of exp2 / log2) -> + (V + 8) u (|L| + 1)
  dS entry   exp(z - L) is off by its own size times (e_z + e_L); a target adds its p times 4 u; then one rounding: half a step of
             the 16-bit type, its square in two planes (up to 256 rows), 2^-22 for fp32's two fp16 planes; fp16 has no step below
             2^-24, and dS is scaled to 2^13 at most: 2^-36 of the largest |g T|
  gradients  the entries' errors times the other factor, plus (c + n u) of the sum of sizes, plus half a step of the output's type
"""
import os

import pytest
import torch

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _inputs(dtype, R, V, K, bias=True, seed=0, device="cuda", spread=2.0):
    g = torch.Generator().manual_seed(seed)
    dt = DT[dtype]
    h = torch.randn(R, K, generator=g).to(dt).to(device)
    w = (torch.randn(V, K, generator=g) * (spread / K ** 0.5)).to(dt).to(device)
    b = (torch.randn(V, generator=g) * 0.5).to(dt).to(device) if bias else None
    return h, w, b, g


def _oracle(h, w, b, ids, p, T, g):
    """Losses, gradients and their error bounds in fp64; ids / p (R, S): targets (p rows of 0: the row does not count); g (R,)."""
    K, V, dt = h.shape[1], w.shape[0], h.dtype
    H, W = h.double(), w.double()
    z = H @ W.t()
    size = H.abs() @ W.abs().t()
    if b is not None:
        z = z + b.double()
        size = size + b.double().abs()
    z, size = z / T, size / T
    c = 3 * 2.0 ** -22 if dt == torch.float32 else 0.0
    e_z = (c + K * U) * size + 4 * U * z.abs().nan_to_num(posinf=0.0)
    L = torch.logsumexp(z, 1)
    live = (p.sum(1) > 0).double()
    slot = ids.clamp(min=0)
    e_max = e_z.max(1)[0]
    e_L = e_max + (V + 8) * U * (L.abs() + 1)
    zt = z.gather(1, slot)
    logp = torch.where(p > 0, p.log(), torch.zeros_like(p))
    loss = live * T * T * (p * (logp - torch.where(p > 0, zt, torch.zeros_like(zt)) + L[:, None])).sum(1)
    e_loss = live * T * T * (e_max + e_L + 16 * U * ((p * (logp.abs() + torch.where(p > 0, zt, torch.zeros_like(zt)).abs())).sum(1)
                                                        + L.abs() + 1) + ids.shape[1] * U)
    q = (z - L[:, None]).exp()
    target = torch.zeros_like(q).scatter_add_(1, slot, torch.where(ids >= 0, p, torch.zeros_like(p)))
    gt = (g.double() * T * live)[:, None]
    dS = gt * (q - target)
    rnd = 2.0 ** -22 if dt == torch.float32 else HALF[dt] ** 2 if h.shape[0] <= 256 else HALF[dt]
    e_S = gt.abs() * (q * (e_z + e_L[:, None]) * 1.01 + 8 * U * (target + q)) + 4 * U * dS.abs()
    e_S = e_S + rnd * (dS.abs() + e_S) + (2.0 ** -36 * gt.abs().max() if dt != torch.bfloat16 else 0.0)
    out = {"loss": (loss, e_loss)}

    def product(x, ex, y, n):
        v = x @ y
        e = (ex @ y.abs()) + (c + n * U) * (x.abs() @ y.abs())
        return v, e + HALF[dt] * (v.abs() + e) + 2.0 ** -140
    out["d_hidden"] = product(dS, e_S, W, V)
    out["d_weight"] = product(dS.t(), e_S.t(), H, h.shape[0])
    if b is not None:
        # a stage of at least 32 rows is summed first, its 64 values off by 64 u at most, then the stages; few rows: every fourth row
        v, e = dS.sum(0), e_S.sum(0) + ((h.shape[0] / 32 if h.shape[0] > 4096 else h.shape[0] / 4) + 68) * U * dS.abs().sum(0)
        out["d_bias"] = (v, e + HALF[b.dtype] * (v.abs() + e) + 2.0 ** -140)
    return out


def _hold(got, want, what):
    v, e = want
    d = (got.double() - v).abs()
    if got.dtype == torch.float16:
        e = e + 2.0 ** -25                        # fp16 has no finer step
    bad = ~(d <= e)
    assert not bool(bad.any()), "%s: %d of %d over the bound, worst %.3g of a bound of %.3g" % (
        what, int(bad.sum()), d.numel(), float(d[bad].max()), float(e.expand_as(d)[bad][d[bad].argmax()]))


def _leaves(h, w, b):
    return [t.detach().requires_grad_() if t is not None else None for t in (h, w, b)]      # (a clone would lose the strides)


def _run_ce(h, w, b, labels, g, ignore=-1):
    from gridmm_amd import vocab
    hl, wl, bl = _leaves(h, w, b)
    loss = vocab.vocab_cross_entropy(hl, wl, labels, bias=bl, ignore_index=ignore)
    loss.backward(g)
    got = {"loss": loss.detach(), "d_hidden": hl.grad, "d_weight": wl.grad}
    if b is not None:
        got["d_bias"] = bl.grad
    return got


def _check_ce(h, w, b, labels, g, ignore=-1):
    got = _run_ce(h, w, b, labels, g, ignore)
    p = (labels != ignore).double()[:, None]
    want = _oracle(h, w, b, torch.where(labels == ignore, torch.zeros_like(labels), labels).long()[:, None], p, 1.0, g)
    for k, v in want.items():
        assert got[k].dtype == (torch.float32 if k == "loss" else w.dtype if k != "d_bias" else b.dtype)
        _hold(got[k], v, k)
    return got


CE = [("fp32", 1, 1, 1), ("fp32", 1, 300, 64), ("bf16", 1, 257, 64), ("fp16", 3, 1000, 72), ("fp32", 37, 1000, 256), ("bf16", 129, 511, 128),
      ("fp16", 64, 256, 64), ("fp32", 200, 777, 33), ("bf16", 65, 1025, 200), ("fp16", 130, 2049, 96), ("fp32", 257, 513, 768),
      ("bf16", 300, 70000, 64), ("fp32", 300, 70000, 64), ("bf16", 7, 40000, 64)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,R,V,K", CE)
@pytest.mark.parametrize("bias", [False, True])
def test_cross_entropy_and_its_gradients(dtype, R, V, K, bias):
    h, w, b, g = _inputs(dtype, R, V, K, bias, seed=R + V + K)
    labels = torch.randint(0, V, (R,), generator=g)
    if R > 2:
        labels[torch.rand(R, generator=g) < 0.3] = -1
    labels[0], labels[-1] = 0, V - 1
    _check_ce(h, w, b, labels.cuda(), (torch.rand(R, generator=g) - 0.3).cuda())


# over 6e8 operations and 32 rows: the kernels on packed tiles (the smaller ones above take those for few rows)
CE_TILES = [("fp32", 33, 30011, 320), ("bf16", 17, 40000, 513), ("fp16", 129, 4099, 600), ("fp32", 257, 1300, 1000), ("bf16", 511, 3001, 264),
            ("fp16", 1025, 1025, 320), ("fp32", 700, 20001, 33), ("bf16", 2000, 700, 256), ("fp16", 300, 33000, 65), ("fp32", 129, 3000, 800)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,R,V,K", CE_TILES)
@pytest.mark.parametrize("bias", [False, True])
def test_cross_entropy_on_tiles(dtype, R, V, K, bias):
    test_cross_entropy_and_its_gradients(dtype, R, V, K, bias)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,R,V,K", [("fp32", 60001, 70, 40), ("bf16", 100000, 129, 64)])
def test_cross_entropy_of_very_many_rows(dtype, R, V, K):
    h, w, b, g = _inputs(dtype, R, V, K, True, seed=6)
    labels = torch.randint(0, V, (R,), generator=g)
    labels[torch.rand(R, generator=g) < 0.1] = -1
    _check_ce(h, w, b, labels.cuda(), (torch.rand(R, generator=g) / R).cuda())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("drop", [0.0, 0.98])
def test_cross_entropy_over_several_pieces(dtype, drop):
    """More columns than one piece of dS holds (512 MB of 16-bit values), a narrower last piece; few of the rows count in one run."""
    R, V, K = 9100, 33001, 72
    h, w, b, g = _inputs(dtype, R, V, K, True, seed=5)
    labels = torch.randint(0, V, (R,), generator=g)
    labels[torch.rand(R, generator=g) < drop] = -1
    _check_ce(h, w, b, labels.cuda(), (torch.rand(R, generator=g) / R).cuda())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("V,K", [(300, 64), (30000, 192)])
def test_cross_entropy_of_rows_that_are_all_ignored(dtype, V, K):
    h, w, b, _ = _inputs(dtype, 70, V, K)
    h[3] = float("nan")                            # an ignored row's values are never read into a result
    got = _run_ce(h, w, b, torch.full((70,), -100, device="cuda"), torch.ones(70, device="cuda"), ignore=-100)
    for v in got.values():
        assert bool((v == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("V,K", [(500, 64), (40000, 256)])
def test_ignored_rows_may_hold_anything(V, K):
    h, w, b, g = _inputs("fp32", 40, V, K)
    labels = torch.randint(0, V, (40,), generator=g).cuda()
    labels[::3] = -1
    clean = _run_ce(h, w, b, labels, torch.ones(40, device="cuda"))
    h[0], h[3] = float("nan"), 3.0e38
    dirty = _run_ce(h, w, b, labels, torch.ones(40, device="cuda"))
    for k in clean:
        assert torch.equal(clean[k], dirty[k]), k


@pytest.mark.gpu
@pytest.mark.parametrize("index", [torch.int64, torch.int32])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("R,V,K", [(50, 333, 64), (200, 12001, 128)])
def test_cross_entropy_of_strided_operands(dtype, index, R, V, K):
    """Rows of a wider matrix, off a 16-byte boundary; a transposed weight; a batch of sequences."""
    g = torch.Generator().manual_seed(3)
    big = torch.randn(R, K + 19, generator=g).to(DT[dtype]).cuda()
    wt = (torch.randn(K, V, generator=g) / 4).to(DT[dtype]).cuda()
    wbig = (torch.randn(V, 2 * K + 5, generator=g) / 4).to(DT[dtype]).cuda()
    labels = torch.randint(0, V, (R,), generator=g).to(index).cuda()
    gr = torch.rand(R, generator=g).cuda()
    for h, w in ((big[:, 3:3 + K], wbig[:, 7:7 + K]), (big[:, :K], wt.t()), (big.view(-1)[:R * K].view(R, K), wbig[:, :K])):
        _check_ce(h, w, None, labels, gr)
    from gridmm_amd import vocab
    w = wt.t().contiguous()
    h3 = big[:, :K].contiguous().view(5, R // 5, K)
    a = vocab.vocab_cross_entropy(h3, w, labels.view(5, R // 5))
    assert a.shape == (5, R // 5) and torch.equal(a.view(-1), vocab.vocab_cross_entropy(h3.reshape(R, K), w, labels))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("R,V,K", [(20, 300, 64), (2000, 300, 520), (2000, 320, 512)])
def test_rows_of_weight_far_apart(dtype, R, V, K):
    """2^23 elements and more from one row of W to the next: 32 bits of bytes do not reach over a tile's rows."""
    g = torch.Generator().manual_seed(8)
    ld = 2 ** 23 + 64
    far = torch.empty(V * ld, dtype=DT[dtype], device="cuda").as_strided((V, K), (ld, 1))
    far.copy_((torch.randn(V, K, generator=g) / 8).to(DT[dtype]))
    h = torch.randn(R, K, generator=g).to(DT[dtype]).cuda()
    _check_ce(h, far, None, torch.randint(0, V, (R,), generator=g).cuda(), torch.rand(R, generator=g).cuda())


@pytest.mark.gpu
@pytest.mark.parametrize("V", [200, 40000])
def test_single_rows_and_broadcast_rows(V):
    """A single row may carry any stride, and the same row may stand for many."""
    from gridmm_amd import vocab
    h, w, b, g = _inputs("fp32", 1, V, 128)
    y = torch.tensor([3], device="cuda")
    a = vocab.vocab_cross_entropy(h, w, y, bias=b)
    assert torch.equal(a, vocab.vocab_cross_entropy(h[0].as_strided((1, 128), (0, 1)), w, y, bias=b))
    ids, t = torch.tensor([[1, 5, 9]], device="cuda"), torch.tensor([[0.5, 1.0, -1.0]], device="cuda")
    c = vocab.vocab_distillation(h, w, ids, t, bias=b)
    assert torch.equal(c, vocab.vocab_distillation(h, w, ids[0].as_strided((1, 3), (0, 1)), t[0].as_strided((1, 3), (0, 1)), bias=b))
    x = h @ w.t()
    for one, two in zip(vocab.top_logits(x, 4), vocab.top_logits(x[0].as_strided((1, V), (0, 1)), 4)):
        assert torch.equal(one, two)
    hl = h.clone().requires_grad_()
    many = vocab.vocab_cross_entropy(hl.expand(70, 128), w, y.expand(70), bias=b)
    assert bool((many == many[0]).all())
    many.sum().backward()
    _check_ce(h.expand(70, 128).contiguous(), w, b, y.expand(70).contiguous(), torch.ones(70, device="cuda"))
    hf = h.expand(70, 128).contiguous().requires_grad_()
    vocab.vocab_cross_entropy(hf, w, y.expand(70).contiguous(), bias=b).sum().backward()
    assert torch.equal(hl.grad, hf.grad.sum(0, keepdim=True))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("V,K", [(600, 64), (40000, 256)])
def test_bias_of_minus_infinity_masks_a_column(dtype, V, K):
    h, w, b, g = _inputs(dtype, 33, V, K)
    labels = torch.randint(0, 300, (33,), generator=g).cuda()
    b[300:] = float("-inf")                        # whole tiles without a live column
    w[400] = 60.0
    hl, wl, bl = _leaves(h, w, b)
    from gridmm_amd import vocab
    gr = torch.rand(33, generator=g).cuda()
    loss = vocab.vocab_cross_entropy(hl, wl, labels, bias=bl)
    loss.backward(gr)
    want = _oracle(h, w[:300], b[:300], labels[:, None], torch.ones(33, 1, device="cuda", dtype=torch.float64), 1.0, gr)
    for k, t in (("loss", loss.detach()), ("d_hidden", hl.grad), ("d_weight", wl.grad[:300]), ("d_bias", bl.grad[:300])):
        v, e = want[k]
        _hold(t, (v, e), k)                        # (w[400] sets the scale of the fp32 planes, which changes their range and not their 22 bits)
    assert bool((wl.grad[300:] == 0).all()) and bool((bl.grad[300:] == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("V,K", [(600, 64), (40000, 256)])
def test_bias_of_the_lowest_finite_value(dtype, V, K):
    """A column masked with the type's lowest number: nothing for the rows that do not aim at it, a huge but finite loss for those that
    do (the number over log 2 is no longer a fp32 number)."""
    h, w, b, g = _inputs(dtype, 33, V, K)
    b[10:300] = torch.finfo(b.dtype).min
    labels = torch.randint(300, V, (33,), generator=g).cuda()
    labels[::4], labels[1] = 17, 3
    got = _check_ce(h, w, b, labels, torch.rand(33, generator=g).cuda())
    assert bool(torch.isfinite(got["loss"]).all()) and float(got["loss"][0]) > 6e4
    ids = torch.stack([torch.randperm(V, generator=g)[:7] for _ in range(33)])
    ids[0, 0] = 17
    _check_kd(h, w, b, ids.cuda(), torch.randn(33, 7, generator=g).cuda(), torch.rand(33, generator=g).cuda(), 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("R,V,K", [(20, 100, 64), (40, 40000, 256)])
def test_a_label_outside_the_vocabulary_spoils_its_row_and_nothing_else(R, V, K):
    h, w, b, g = _inputs("fp32", R, V, K)
    labels = torch.randint(0, V, (R,), generator=g).cuda()
    good = _run_ce(h, w, b, labels, torch.ones(R, device="cuda"))
    for bad in (V, -2, 2 ** 31 - 1, -2 ** 40):
        lab = labels.clone()
        lab[7] = bad
        got = _run_ce(h, w, b, lab, torch.ones(R, device="cuda"))
        keep = torch.arange(R, device="cuda") != 7
        assert bool(torch.isnan(got["loss"][7])) and torch.equal(got["loss"][keep], good["loss"][keep])
        assert bool(torch.isnan(got["d_hidden"][7]).all()) and torch.equal(got["d_hidden"][keep], good["d_hidden"][keep])
        assert bool(torch.isnan(got["d_bias"]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("R,V,K", [(20, 100, 64), (40, 40000, 256)])
def test_a_row_of_nan_or_infinity_stays_its_own(R, V, K):
    for bad in (float("nan"), float("inf")):
        h, w, b, g = _inputs("fp32", R, V, K)
        labels = torch.randint(0, V, (R,), generator=g).cuda()
        good = _run_ce(h, w, b, labels, torch.ones(R, device="cuda"))
        h[5, 3] = bad
        got = _run_ce(h, w, b, labels, torch.ones(R, device="cuda"))
        keep = torch.arange(R, device="cuda") != 5
        assert bool(torch.isnan(got["loss"][5]))
        scale = good["loss"][keep].abs().max()
        assert float((got["loss"][keep] - good["loss"][keep]).abs().max()) <= 8 * U * K * float(scale + 8)


def _kd_inputs(dtype, R, V, K, S, seed):
    h, w, b, g = _inputs(dtype, R, V, K, True, seed)
    ids = torch.stack([torch.randperm(V, generator=g)[:S] for _ in range(R)])
    t = torch.randn(R, S, generator=g) * 3
    return h, w, b, ids, t, g


def _teacher(ids, t, T):
    t = torch.where(ids >= 0, t.double() / T, torch.full_like(t.double(), float("-inf")))
    p = torch.softmax(t, 1)
    return torch.nan_to_num(p)


def _check_kd(h, w, b, ids, t, g, T):
    from gridmm_amd import vocab
    hl, wl, bl = _leaves(h, w, b)
    loss = vocab.vocab_distillation(hl, wl, ids, t, bias=bl, temperature=T)
    loss.backward(g)
    want = _oracle(h, w, b, ids.long(), _teacher(ids, t, T), T, g)
    got = {"loss": loss.detach(), "d_hidden": hl.grad, "d_weight": wl.grad, "d_bias": bl.grad}
    for k, v in want.items():
        _hold(got[k], v, k)


KD = [("fp32", 300, 9001, 130, 17, 2.0), ("bf16", 200, 20001, 128, 300, 1.0), ("fp16", 1030, 2500, 200, 5, 0.5), ("fp32", 60, 30522, 256, 64, 1.0),
      ("fp32", 1, 1, 64, 1, 1.0), ("fp32", 5, 300, 64, 8, 2.0), ("bf16", 130, 1000, 128, 32, 1.0), ("fp16", 77, 513, 72, 100, 0.5),
      ("fp32", 300, 2000, 100, 17, 4.0), ("bf16", 3, 40000, 64, 256, 1.5), ("fp32", 64, 256, 64, 256, 1.0), ("fp32", 16, 30522, 64, 8200, 1.0),
      # many slots of long rows: the scores at the targets out of the score tiles (128 x 128, 256 x 256, two pieces of W)
      ("bf16", 700, 3001, 1024, 100, 1.5), ("fp16", 2100, 11000, 520, 70, 0.5), ("fp32", 300, 5000, 1030, 120, 2.0), ("fp32", 300, 62000, 2200, 60, 2.0),
      ("fp32", 2100, 11003, 512, 40, 1.0)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,R,V,K,S,T", KD)
def test_distillation_and_its_gradients(dtype, R, V, K, S, T):
    h, w, b, ids, t, g = _kd_inputs(dtype, R, V, K, S, seed=R + S)
    if R > 4:
        ids[torch.rand(R, S, generator=g) < 0.2] = -1
        ids[1] = -1                                    # a row without a target
        t[2] = float("-inf")                           # a row whose teacher says nothing
        t[3, 0] = float("-inf")
    _check_kd(h, w, b, ids.cuda(), t.cuda(), torch.rand(R, generator=g).cuda(), T)


@pytest.mark.gpu
@pytest.mark.parametrize("V,K", [(90, 64), (40000, 256)])
def test_distillation_where_ids_repeat_and_are_int32_columns_of_a_wider_table(V, K):
    h, w, b, ids, t, g = _kd_inputs("fp32", 40, V, K, 12, seed=1)
    ids = torch.randint(0, 5, (40, 15), generator=g)
    t = torch.randn(40, 20, generator=g)
    _check_kd(h, w, b, ids.int().cuda()[:, 2:14], t.cuda()[:, 3:15], torch.rand(40, generator=g).cuda(), 1.0)


@pytest.mark.gpu
def test_distillation_from_many_slots_where_ids_repeat_and_columns_are_masked():
    """The scores at the targets out of the score tiles: repeated ids, all of a row's ids in one block, int32, the lowest bias."""
    h, w, b, g = _inputs("fp32", 600, 2000, 1024, True, 2)
    b[40:60] = torch.finfo(torch.float32).min
    ids = torch.randint(0, 2000, (600, 64), generator=g)
    ids[1] = torch.randint(70, 75, (64,), generator=g)
    ids[2] = 1999
    ids[3, ::2], ids[3, 1::2] = -1, 50
    _check_kd(h, w, b, ids.int().cuda(), torch.randn(600, 64, generator=g).cuda(), torch.rand(600, generator=g).cuda(), 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("R,V,K,S", [(10, 300, 64, 4), (40, 40000, 256, 4), (600, 2000, 1024, 80)])
def test_distillation_of_an_id_past_the_vocabulary(R, V, K, S):
    from gridmm_amd import vocab
    h, w, b, ids, t, g = _kd_inputs("bf16", R, V, K, S, seed=1)
    good = vocab.vocab_distillation(h, w, ids.cuda(), t.cuda(), bias=b)
    ids[4, 2] = V
    got = vocab.vocab_distillation(h, w, ids.cuda(), t.cuda(), bias=b)
    keep = torch.arange(R, device="cuda") != 4
    assert bool(torch.isnan(got[4])) and torch.equal(got[keep], good[keep])


@pytest.mark.gpu
def test_one_slot_at_temperature_one_is_cross_entropy():
    from gridmm_amd import vocab
    h, w, b, g = _inputs("fp32", 50, 700, 128)
    labels = torch.randint(0, 700, (50,), generator=g).cuda()
    a = vocab.vocab_cross_entropy(h, w, labels, bias=b)
    k = vocab.vocab_distillation(h, w, labels[:, None], torch.randn(50, 1, device="cuda"), bias=b)
    assert float((a - k).abs().max()) <= 4 * U * float(a.abs().max() + 1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_gradients_against_differences(dtype):
    """Central differences of the fp32 losses along random directions: step d, error of the difference O(d^2) + noise / d."""
    from gridmm_amd import vocab
    R, V, K, d = 24, 200, 64, 2.0 ** -6
    h, w, b, g = _inputs("fp32", R, V, K, True, seed=9, spread=1.0)
    ids = torch.stack([torch.randperm(V, generator=g)[:6] for _ in range(R)]).cuda()
    t = torch.randn(R, 6, generator=g).cuda()
    labels = torch.randint(0, V, (R,), generator=g).cuda()
    cast = DT[dtype]
    for f in (lambda a, m, c: vocab.vocab_cross_entropy(a, m, labels, bias=c),
              lambda a, m, c: vocab.vocab_distillation(a, m, ids, t, bias=c, temperature=2.0)):
        hl, wl, bl = _leaves(h.to(cast), w.to(cast), b.to(cast))
        f(hl, wl, bl).sum().backward()
        for leaf in (hl, wl, bl):
            u = torch.randn(leaf.shape, generator=g).cuda()
            u = u / u.norm() * d
            args = [x.detach().float() for x in (hl, wl, bl)]
            i = [x is leaf for x in (hl, wl, bl)].index(True)
            up, dn = list(args), list(args)
            up[i], dn[i] = args[i] + u, args[i] - u
            slope = float((f(*up).double().sum() - f(*dn).double().sum()) / 2)
            want = float((leaf.grad.double() * u.double()).sum())
            # third derivative of a log-sum-exp along a step of size s (in scores): s^3 / 3 a row at most; noise: R losses of ~8 off by 2^-20
            step = float((u.double().norm()) * max(float(h.double().norm(dim=1).max()), float(w.double().norm(dim=1).max()), 1.0))
            bound = R * step ** 3 + R * 8 * 2.0 ** -19 + (2 * HALF[cast] if dtype != "fp32" else 2.0 ** -18) * float((leaf.grad.double().abs() * u.double().abs()).sum())
            assert abs(slope - want) <= bound, (slope, want, bound)


@pytest.mark.gpu
@pytest.mark.parametrize("R,V,K", [(30, 400, 64), (40, 40000, 256)])
def test_only_the_gradients_that_are_asked_for(R, V, K):
    from gridmm_amd import vocab
    h, w, b, g = _inputs("fp32", R, V, K)
    labels = torch.randint(0, V, (R,), generator=g).cuda()
    full = _run_ce(h, w, b, labels, torch.ones(R, device="cuda"))
    for mask in range(1, 8):
        ts = [t.detach().clone().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate((h, w, b))]
        vocab.vocab_cross_entropy(ts[0], ts[1], labels, bias=ts[2]).sum().backward()      # (a gradient of stride 0)
        for i, k in enumerate(("d_hidden", "d_weight", "d_bias")):
            if mask >> i & 1:
                assert torch.equal(ts[i].grad, full[k]), (mask, k)
            else:
                assert ts[i].grad is None


@pytest.mark.gpu
@pytest.mark.parametrize("R,V,K", [(20, 500, 64), (600, 2000, 100), (600, 30000, 100)])
def test_without_recording_a_parameter_is_a_plain_tensor(R, V, K):
    """Under no_grad leaves that want gradients give what plain tensors give, bit for bit, and nothing is kept for a backward."""
    from gridmm_amd import vocab
    h, w, b, g = _inputs("fp32", R, V, K)
    labels = torch.randint(0, V, (R,), generator=g).cuda()
    want = vocab.vocab_cross_entropy(h, w, labels, bias=b)
    hl, wl, bl = _leaves(h, w, b)
    with torch.no_grad():
        got = vocab.vocab_cross_entropy(hl, wl, labels, bias=bl)
    assert torch.equal(got, want) and not got.requires_grad
    recorded = vocab.vocab_cross_entropy(hl, wl, labels, bias=bl)
    # the two sets of kernels: fp32 products and sums, or two fp16 planes of each operand (_oracle's e_z, twice)
    size = (h.double().abs() @ w.double().abs().t() + b.double().abs()).max(1)[0]
    bound = 2 * (2 * (3 * 2.0 ** -22 + K * U) * size + (V + 32) * U * (want.double().abs() + size + 1))
    assert bool(((recorded.detach().double() - want.double()).abs() <= bound).all())


@pytest.mark.gpu
@pytest.mark.parametrize("V", [3000, 30000])
def test_runs_repeat_bit_for_bit_and_leave_their_inputs(V):
    h, w, b, g = _inputs("bf16", 300, V, 128)
    labels = torch.randint(0, V, (300,), generator=g).cuda()
    gr = torch.rand(300, generator=g).cuda()
    copies = [t.clone() for t in (h, w, b, labels, gr)]
    first = _run_ce(h, w, b, labels, gr)
    for _ in range(3):
        again = _run_ce(h, w, b, labels, gr)
        for k in first:
            assert torch.equal(first[k], again[k]), k
    for a, c in zip((h, w, b, labels, gr), copies):
        assert torch.equal(a, c)


@pytest.mark.gpu
@pytest.mark.parametrize("V,K", [(500, 64), (40000, 256)])
def test_backward_twice_of_a_retained_graph_with_other_gradients(V, K):
    from gridmm_amd import vocab
    h, w, b, g = _inputs("fp16", 40, V, K)
    labels = torch.randint(0, V, (40,), generator=g).cuda()
    hl, wl, bl = _leaves(h, w, b)
    loss = vocab.vocab_cross_entropy(hl, wl, labels, bias=bl)
    for scale in (1.0, 1e-4, 64.0):
        gr = (torch.rand(40, generator=g) * scale).cuda()
        got = torch.autograd.grad(loss, (hl, wl, bl), gr, retain_graph=True)
        want = _run_ce(h, w, b, labels, gr)
        for x, k in zip(got, ("d_hidden", "d_weight", "d_bias")):
            assert torch.equal(x, want[k])


@pytest.mark.gpu
def test_a_weight_changed_before_the_backward_is_refused():
    from gridmm_amd import vocab
    h, w, b, g = _inputs("fp32", 10, 100, 64)
    hl, wl, bl = _leaves(h, w, b)
    loss = vocab.vocab_cross_entropy(hl, wl, torch.zeros(10, dtype=torch.long, device="cuda"), bias=bl)
    with torch.no_grad():
        wl.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.sum().backward()


@pytest.mark.gpu
def test_no_rows():
    from gridmm_amd import vocab
    h, w, b, _ = _inputs("bf16", 0, 100, 64)
    got = _run_ce(h, w, b, torch.zeros(0, dtype=torch.long, device="cuda"), torch.zeros(0, device="cuda"))
    assert got["loss"].shape == (0,) and got["d_hidden"].shape == (0, 64)
    assert bool((got["d_weight"] == 0).all()) and bool((got["d_bias"] == 0).all())
    v, i, l = vocab.top_logits(torch.zeros(0, 10, device="cuda"), 3)
    assert v.shape == (0, 3) and i.shape == (0, 3) and l.shape == (0,)


@pytest.mark.gpu
@pytest.mark.parametrize("V", [2000, 40000])
def test_on_another_stream(V):
    h, w, b, g = _inputs("fp32", 100, V, 128)
    labels = torch.randint(0, V, (100,), generator=g).cuda()
    gr = torch.rand(100, generator=g).cuda()
    want = _run_ce(h, w, b, labels, gr)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = _run_ce(h, w, b, labels, gr)
    torch.cuda.current_stream().wait_stream(st)
    for k in want:
        assert torch.equal(want[k], got[k])


@pytest.mark.gpu
@pytest.mark.parametrize("V", [1500, 15000])
def test_captured_step_replays_with_other_labels_and_other_counts(V):
    """Forward and backward in one hipGraph; between the replays the labels (and with them the number of rows that count) change and
    eager work of the same operators runs."""
    from gridmm_amd import vocab
    h, w, b, g = _inputs("fp32", 300, V, 128)
    hl, wl, bl = _leaves(h, w, b)
    labels = torch.randint(0, V, (300,), generator=g).cuda()
    gr = torch.rand(300, generator=g).cuda()

    def step():
        loss = vocab.vocab_cross_entropy(hl, wl, labels, bias=bl)
        return (loss,) + torch.autograd.grad(loss, (hl, wl, bl), gr)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(st)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for drop in (0.0, 0.5, 1.0, 0.1):
        new = torch.randint(0, V, (300,), generator=g)
        new[torch.rand(300, generator=g) < drop] = -1
        labels.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        want = _run_ce(h, w, b, labels, gr)
        for x, k in zip(out, ("loss", "d_hidden", "d_weight", "d_bias")):
            assert torch.equal(x, want[k]), (drop, k)


@pytest.mark.gpu
@pytest.mark.parametrize("V", [1500, 30000])
def test_two_calls_at_once_and_two_captured_ones(V):
    """Calls on two streams side by side, then each captured (one memory pool) and both replayed in turn: every result is the one that a
    call alone gives."""
    from gridmm_amd import vocab
    sets = []
    for seed in (1, 2):
        h, w, b, g = _inputs("bf16", 300, V, 192, True, seed)
        labels, gr = torch.randint(0, V, (300,), generator=g).cuda(), torch.rand(300, generator=g).cuda()
        sets.append((_leaves(h, w, b), labels, gr, _run_ce(h, w, b, labels, gr)))

    def step(i):
        (hl, wl, bl), labels, gr, _ = sets[i]
        loss = vocab.vocab_cross_entropy(hl, wl, labels, bias=bl)
        return (loss,) + torch.autograd.grad(loss, (hl, wl, bl), gr)

    def same(i, out):
        for x, k in zip(out, ("loss", "d_hidden", "d_weight", "d_bias")):
            assert torch.equal(x, sets[i][3][k]), (i, k)
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(3):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                outs[i].append(step(i))
    torch.cuda.synchronize()
    for i in (0, 1):
        for out in outs[i]:
            same(i, out)
    graphs, pool = [], None
    for i in (0, 1):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i], pool=pool):
            outs[i] = step(i)
        pool = graphs[0].pool()
    for order in ((0, 1), (0, 1, 0), (0, 1, 0, 1)):
        for i in order:
            graphs[i].replay()
            torch.cuda.synchronize()
            same(i, outs[i])
            same(1 - i, step(1 - i))                   # eager work between the replays


# ---- top logits ----
def _top_oracle(x, k):
    key = x.float().cpu()
    key = torch.where(torch.isnan(key), torch.full_like(key, float("inf")), key)
    nan = torch.isnan(x.float().cpu())
    out = []
    for r in range(x.shape[0]):
        order = sorted(range(x.shape[1]), key=lambda j: (not bool(nan[r, j]), -float(key[r, j]), j))[:k]
        out.append(order)
    return torch.tensor(out, dtype=torch.int64)


def _check_top(x, k):
    from gridmm_amd import vocab
    values, ids, lse = vocab.top_logits(x, k)
    want = _top_oracle(x, k)
    assert torch.equal(ids.cpu(), want)
    assert torch.equal(torch.nan_to_num(values, nan=7.0), torch.nan_to_num(x.gather(1, want.to(x.device)), nan=7.0))
    z = torch.logsumexp(x.double(), 1)
    fine = torch.isfinite(z)
    assert torch.equal(torch.isnan(z), torch.isnan(lse)) and torch.equal(z[~fine & ~torch.isnan(z)].float(), lse[~fine & ~torch.isnan(z)])
    # a sum of V fp32 exponentials in pieces, each off by 2 steps of exp and one of its argument
    bound = (x.shape[1] ** 0.5 + 16) * U * (z[fine].abs() + x[fine].double().nan_to_num(neginf=0.0).abs().amax(1) + 1)
    assert bool(((lse[fine].double() - z[fine]).abs() <= bound).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("R,V,k", [(1, 1, 1), (1, 5, 5), (3, 64, 7), (7, 1000, 1), (2, 1025, 1024), (5, 4099, 100), (1, 70001, 256),
                                   (2, 30522, 32), (300, 257, 16)])
def test_top_logits(dtype, R, V, k):
    g = torch.Generator().manual_seed(V + k)
    _check_top((torch.randn(R, V, generator=g) * 3).to(DT[dtype]).cuda(), k)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_top_logits_of_rows_that_are_hard_to_select_from(dtype):
    dt, V = DT[dtype], 9001
    rows = [torch.zeros(V), torch.arange(V) / 64.0, -torch.arange(V) / 64.0, torch.full((V,), float("-inf")), torch.full((V,), float("inf"))]
    few = torch.full((V,), float("-inf"))
    few[[17, 4000, 8999]] = torch.tensor([1.0, -3.0, 1.0])
    signed = torch.zeros(V)
    signed[::2] = -0.0
    nan = torch.randn(V, generator=torch.Generator().manual_seed(0))
    nan[[5, 7000]] = float("nan")
    big = torch.randn(V, generator=torch.Generator().manual_seed(1)) * 1e4
    two = torch.where(torch.arange(V) % 3 == 0, 2.0, 1.0)
    x = torch.stack(rows + [few, signed, nan, big, two]).to(dt).cuda()
    for k in (1, 3, 64, 1000):
        _check_top(x, k)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("V,k,R", [(131071, 64, 1), (131072, 1000, 3), (20000, 1024, 7), (8193, 200, 40), (50021, 1, 5), (50021, 16, 700)])
def test_top_logits_of_long_rows(dtype, V, k, R):
    """Rows cut into segments or read by one workgroup in many chunks; rising rows, where every value enters, and constant ones."""
    from gridmm_amd import vocab
    g = torch.Generator().manual_seed(V)
    x = torch.randn(R, V, generator=g) * 3
    x[0] = torch.arange(V) / 512.0
    if R > 1:
        x[1] = 1.5
        x[2, : V - 5] = float("-inf")
    x = x.to(DT[dtype]).cuda()
    values, ids, lse = vocab.top_logits(x, k)
    want, order = x.float().sort(dim=1, descending=True, stable=True)
    assert torch.equal(ids, order[:, :k]) and torch.equal(values.float(), want[:, :k])
    z = torch.logsumexp(x.double(), 1)
    assert bool(((lse.double() - z).abs() <= (V ** 0.5 + 16) * U * (z.abs() + want[:, 0].double().abs() + 1)).all())


@pytest.mark.gpu
def test_top_logits_of_rows_of_a_wider_matrix_and_of_a_batch():
    from gridmm_amd import vocab
    g = torch.Generator().manual_seed(2)
    x = torch.randn(6, 1000, generator=g).bfloat16().cuda()
    _check_top(x[:, 3:990], 20)
    _check_top(x.t()[:500, :5].t(), 9)
    v, i, l = vocab.top_logits(x.view(2, 3, 1000), 4)
    v2, i2, l2 = vocab.top_logits(x, 4)
    assert v.shape == i.shape == (2, 3, 4) and l.shape == (2, 3)
    assert torch.equal(v.view(6, 4), v2) and torch.equal(i.view(6, 4), i2) and torch.equal(l.view(6), l2)
    v1, i1, l1 = vocab.top_logits(x[0], 4)
    assert torch.equal(v1, v2[0]) and torch.equal(i1, i2[0]) and torch.equal(l1, l2[0])


@pytest.mark.gpu
def test_teacher_to_student():
    """The three together, as they are used: a teacher's scores, its top logits, the student's two losses in one backward."""
    from gridmm_amd import vocab
    R, V, K, k, T = 90, 3000, 128, 20, 2.0
    h, w, b, g = _inputs("fp32", R, V, K, True, seed=4)
    teacher = (torch.randn(R, K, generator=g).cuda() + 0.5 * h) @ w.t()
    values, ids, lse = vocab.top_logits(teacher, k)
    assert bool((lse >= values[:, 0]).all())
    labels = torch.randint(0, V, (R,), generator=g).cuda()
    hl, wl, bl = _leaves(h, w, b)
    loss = vocab.vocab_cross_entropy(hl, wl, labels, bias=bl).mean() + 0.5 * vocab.vocab_distillation(hl, wl, ids, values, bias=bl,
                                                                                                      temperature=T).mean()
    loss.backward()
    one = torch.ones(R, 1, device="cuda", dtype=torch.float64)
    a = _oracle(h, w, b, labels[:, None], one, 1.0, torch.full((R,), 1.0 / R, device="cuda"))
    c = _oracle(h, w, b, ids, _teacher(ids, values, T), T, torch.full((R,), 0.5 / R, device="cuda"))
    for name, t in (("d_hidden", hl.grad), ("d_weight", wl.grad), ("d_bias", bl.grad)):
        v = a[name][0] + c[name][0]
        _hold(t, (v, (a[name][1] + c[name][1]) * 1.001 + 2 * U * v.abs()), name)


# ---- the masked-token head ----
def _mlm_model():
    from conftest import load_golden
    from test_hip_pretrain import _model
    return _model(load_golden("pretrain_reduced.npz"))


def _mlm_batch():
    from gridmm_amd.synthetic import batch_to
    from oracle import gen_golden
    return batch_to(gen_golden.pretrain_batch("mlm"), "cuda")


@pytest.mark.gpu
def test_masked_token_head_in_pieces_equals_the_head_that_keeps_its_logits():
    """The same losses and gradients as torch's cross entropy of the kept logits, to what that head's three bf16 terms leave: products
    off by 3 2^-17 of |h| |W| (2^-16 with the bias's share); measured against the reference's gradients elsewhere at 5e-3."""
    m = _mlm_model()
    losses, grads = [], []
    for pieces in (False, True):
        m.config.mlm_in_pieces = pieces
        m.zero_grad()
        loss = m(_mlm_batch(), task="mlm", compute_loss=True)
        loss.mean().backward()
        losses.append(loss.detach())
        grads.append({k: p.grad.clone() for k, p in m.named_parameters() if p.grad is not None})
    m.config.mlm_in_pieces = False
    assert losses[0].shape == losses[1].shape and losses[0].dtype == losses[1].dtype
    # |h| <= sqrt(K) (LayerNorm's rows, unit gain up to a factor 2), rows of W of norm |W|: two scores each off by 2^-15 of the product
    w = m.mlm_head.predictions.decoder.weight
    bound = 2 * 2.0 ** -15 * 2 * w.shape[1] ** 0.5 * float(w.detach().norm(dim=1).max()) + 2.0 ** -20 * float(losses[0].abs().max())
    assert float((losses[0] - losses[1]).abs().max()) <= bound
    assert sorted(grads[0]) == sorted(grads[1])
    scale = max(float(g.norm()) for g in grads[0].values())
    for k in grads[0]:
        a, b = grads[0][k].double(), grads[1][k].double()
        tol = 2e-2 if "text_proj" in k else 5e-3      # (text_proj: arg-max routes, see the reference's own gradients)
        assert float((a - b).norm()) <= tol * max(float(a.norm()), 1e-3 * scale), k


@pytest.mark.gpu
def test_masked_token_head_learns_from_a_teacher():
    """Losses and gradients with a teacher's top logits: cross entropy plus the weighted distillation, of the same hidden states."""
    from gridmm_amd import vocab
    m = _mlm_model()
    batch = _mlm_batch()
    other = dict(batch, **m.mlm_teacher(batch, 12))
    n = other["txt_teacher_ids"].shape[0]
    assert other["txt_teacher_ids"].shape == other["txt_teacher_logits"].shape == (n, 12)
    m.config.mlm_in_pieces = True
    plain = m(_mlm_batch(), task="mlm", compute_loss=True)
    m.config.mlm_distill_weight, m.config.mlm_distill_temperature = 0.5, 2.0
    both = m(other, task="mlm", compute_loss=True)
    # the teacher is the student: the distillation is T^2 KL(p over 12 slots || q over everything) = -T^2 log(q's mass on the slots)
    scores = m(_mlm_batch(), task="mlm", compute_loss=False).detach().double() / 2.0
    mass = torch.log_softmax(scores, 1).gather(1, other["txt_teacher_ids"]).logsumexp(1)
    want = plain.detach().double() - 0.5 * 4.0 * mass
    w = m.mlm_head.predictions.decoder.weight
    bound = 8 * 2.0 ** -15 * 2 * w.shape[1] ** 0.5 * float(w.detach().norm(dim=1).max()) + 2.0 ** -18 * float(want.abs().max())
    assert float((both.detach().double() - want).abs().max()) <= bound
    both.mean().backward()
    assert all(torch.isfinite(p.grad).all() for p in m.parameters() if p.grad is not None)
    assert float(m.mlm_head.predictions.bias.grad.abs().max()) > 0


@pytest.mark.gpu
def test_captured_training_step_with_the_head_in_pieces():
    """Optimizer steps of the captured pre-training step equal the eager ones when the masked-token head runs in pieces and learns from
    a teacher: losses, gradient norms and parameters."""
    import copy
    import train_graph_cases as cases
    from gridmm_amd.pretrain_loop import PreTrainer, default_opts
    from gridmm_amd.train_graph import GraphedTrainStep
    model, batches = cases._setup(0.0)
    model.config.mlm_in_pieces = True
    batch = dict(batches["mlm"], **model.mlm_teacher(batches["mlm"], 8))
    ma, mb = copy.deepcopy(model), copy.deepcopy(model)
    ta, tb = PreTrainer(ma, default_opts(warmup_steps=10)), PreTrainer(mb, default_opts(warmup_steps=10))
    for _ in range(2):                                   # what the graphed object runs while it is built: record + warm-up
        ta.train_step(batch, "mlm")
    g = GraphedTrainStep(tb, batch, "mlm")
    for it in range(4):
        cases._compare_step(ta, tb, lambda: ta.train_step(batch, "mlm"), g, it)


# ---- refusals (no kernel runs) ----
def test_refusals_on_the_cpu():
    from gridmm_amd import _lib, vocab
    h, w, y = torch.zeros(4, 8), torch.zeros(10, 8), torch.zeros(4, dtype=torch.long)
    for call in (lambda: vocab.vocab_cross_entropy(h, w, y), lambda: vocab.vocab_distillation(h, w, y[:, None], h[:, :1]),
                 lambda: vocab.top_logits(h, 2)):
        with pytest.raises(_lib.GridmmLibraryError):
            call()


def _descriptor(**over):
    from gridmm_amd import vocab
    d = vocab._Desc()
    d.rows, d.vocab, d.hidden_size, d.slots, d.temperature = 4, 100, 64, 0, 1.0
    d.ld_hidden = d.ld_weight = 64
    for k, v in over.items():
        setattr(d, k, v)
    return d


def test_the_c_entry_refuses_bad_sizes_and_pointers():
    """The library is called without a GPU: every one of these returns before anything is launched."""
    import ctypes
    from gridmm_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        import __graft_entry__ as g
        g.build()
    lib = _lib.load()
    EINVAL = -1
    assert lib.gridmm_vocab_loss_saved_bytes(ctypes.byref(_descriptor())) > 0
    for over in (dict(rows=-1), dict(vocab=0), dict(hidden_size=0), dict(slots=-1), dict(dtype=3), dict(bias_dtype=-1),
                 dict(temperature=0.0), dict(temperature=float("nan")), dict(temperature=float("inf")), dict(temperature=2.0),
                 dict(rows=2 ** 30), dict(vocab=2 ** 27 + 1), dict(hidden_size=2 ** 21), dict(slots=2 ** 17), dict(slots=1, temperature=1e-7),
                 dict(slots=1, temperature=1e7), dict(rows=2 ** 20, vocab=2 ** 20)):
        d = _descriptor(**over)
        assert lib.gridmm_vocab_loss_saved_bytes(ctypes.byref(d)) == 0, over
        assert lib.gridmm_vocab_loss_workspace(ctypes.byref(d), 0) == 0 and lib.gridmm_vocab_loss_workspace(ctypes.byref(d), 1) == 0
        assert lib.gridmm_vocab_loss_fwd(ctypes.byref(d), 256, 256, 1 << 40, 256, 1 << 40, None) == EINVAL
    ok = dict(hidden=256, weight=256, labels=256, rows=1000, vocab=40000)
    n, ws = lib.gridmm_vocab_loss_saved_bytes(ctypes.byref(_descriptor(**ok))), lib.gridmm_vocab_loss_workspace(ctypes.byref(_descriptor(**ok)), 0)
    for over, args in ((dict(hidden=0), (256, 256, n, 256, ws)), (dict(weight=0), (256, 256, n, 256, ws)), (dict(labels=0), (256, 256, n, 256, ws)),
                       (dict(ld_hidden=63), (256, 256, n, 256, ws)), (dict(ld_weight=63), (256, 256, n, 256, ws)),
                       ({}, (0, 256, n, 256, ws)), ({}, (256, 0, n, 256, ws)), ({}, (256, 256, n - 1, 256, ws)),
                       ({}, (256, 256, n, 0, ws)), ({}, (256, 256, n, 256, ws - 1)), ({}, (256, 16, n, 256, ws)), ({}, (256, 256, n, 16, ws)),
                       (dict(slots=4, ids=256, ld_ids=4, ld_teacher=4), (256, 256, 1 << 40, 256, 1 << 40)),
                       (dict(slots=4, ids=256, teacher=256, ld_ids=3, ld_teacher=4), (256, 256, 1 << 40, 256, 1 << 40))):
        assert lib.gridmm_vocab_loss_fwd(ctypes.byref(_descriptor(**{**ok, **over})), *args, None) == EINVAL, (over, args)
    wb = lib.gridmm_vocab_loss_workspace(ctypes.byref(_descriptor(**ok)), 1)
    for over, args in ((dict(forward_only=1), (256, 1 << 40, 256, 1, 256, 0, 0, 256, 1 << 40)), ({}, (256, n, 0, 1, 256, 256, 0, 256, wb)), ({}, (256, n, 256, 1, 0, 0, 0, 256, wb)), ({}, (256, n, 256, -1, 256, 0, 0, 256, wb)),
                       ({}, (256, n, 256, 1, 256, 0, 256, 256, wb)), ({}, (256, n, 256, 1, 256, 0, 0, 256, wb - 1))):
        assert lib.gridmm_vocab_loss_bwd(ctypes.byref(_descriptor(**{**ok, **over})), *args, None) == EINVAL, (over, args)
    for a in ((256, 9, 0, 1, 10, 2), (256, 10, 3, 1, 10, 2), (256, 10, 0, -1, 10, 2), (256, 10, 0, 1, 10, 0), (256, 10, 0, 1, 10, 11),
              (256, 2000, 0, 1, 2000, 1025), (0, 10, 0, 1, 10, 2)):
        assert lib.gridmm_top_logits(*a, 256, 256, 256, 256, 1 << 40, None) == EINVAL, a


@pytest.mark.gpu
def test_the_wrappers_refuse():
    from gridmm_amd import vocab
    h, w, y = torch.zeros(4, 8).cuda(), torch.zeros(10, 8).cuda(), torch.zeros(4, dtype=torch.long).cuda()
    t = torch.zeros(4, 3).cuda()
    ids = torch.zeros(4, 3, dtype=torch.long).cuda()
    for call in (lambda: vocab.vocab_cross_entropy(h.double(), w.double(), y), lambda: vocab.vocab_cross_entropy(h, w.half(), y),
                 lambda: vocab.vocab_cross_entropy(h[:, :7], w, y), lambda: vocab.vocab_cross_entropy(h, w[0], y),
                 lambda: vocab.vocab_cross_entropy(h, w, y[:3]), lambda: vocab.vocab_cross_entropy(h, w, y.float()),
                 lambda: vocab.vocab_cross_entropy(h, w, y, bias=w[:, 0][:9]), lambda: vocab.vocab_cross_entropy(h, w, y, bias=w[:, 0].half()),
                 lambda: vocab.vocab_cross_entropy(h, w[:0], y), lambda: vocab.vocab_cross_entropy(h[:, :0], w[:, :0], y),
                 lambda: vocab.vocab_distillation(h, w, ids, t[:, :2]), lambda: vocab.vocab_distillation(h, w, ids[:3], t[:3]),
                 lambda: vocab.vocab_distillation(h, w, ids, t, temperature=0.0), lambda: vocab.vocab_distillation(h, w, ids, t, temperature=float("nan")),
                 lambda: vocab.vocab_distillation(h, w, ids.float(), t), lambda: vocab.vocab_distillation(h, w, ids, ids),
                 lambda: vocab.vocab_distillation(h, w, ids[:, :0], t[:, :0]),
                 lambda: vocab.vocab_distillation(h, w, ids, t, temperature=1e-7), lambda: vocab.vocab_distillation(h, w, ids, t, temperature=1e7),
                 lambda: vocab.vocab_distillation(h, w, ids[:, :1].expand(4, 2 ** 16 + 1), t[:, :1].expand(4, 2 ** 16 + 1)),
                 lambda: vocab.vocab_cross_entropy(h[:1].expand(2 ** 20 + 1, 8), w, y[:1].expand(2 ** 20 + 1)),
                 lambda: vocab.vocab_cross_entropy(h[:1].expand(2 ** 20, 8), w[:1].expand(2 ** 20, 8), y[:1].expand(2 ** 20)),
                 lambda: vocab.vocab_cross_entropy(h, w[:1].expand(2 ** 27 + 1, 8), y),
                 lambda: vocab.top_logits(h[:1].expand(2 ** 22 + 1, 8), 1), lambda: vocab.top_logits(h[0, :1].expand(1, 2 ** 31), 1),
                 lambda: vocab.top_logits(h, 0), lambda: vocab.top_logits(h, 9), lambda: vocab.top_logits(h.long(), 1),
                 lambda: vocab.top_logits(torch.zeros(2, 3000).cuda(), 1025)):
        with pytest.raises(ValueError):
            call()
