"""The vocabulary losses and top logits where rounding and range decide: many rows of 16 bits, rows the model is sure of, rows of very
different size, upstream gradients far apart, columns that one tile holds, teachers' and masks' extreme values.

Tolerances (u = 2^-24, half a step of fp32; they count roundings as independent, where a bound that adds all of them would hide what is
looked for; the worst-case bounds are those of test_hip_vocab.py):
  score     an fp32 sum of K products whose partial sums stay below m = max |z| + 1 makes K roundings of at most u m each, in no common
            direction: 8 standard deviations are 8 sqrt(K) u m / sqrt(3); two fp16 planes add 3 2^-22 of each term: less than that again.
            e_z = 8 sqrt(K) u m
  loss      a difference of two such scores, and a sum of positive terms that agree to e_z: 3 e_z
  q = exp(z - L) is off by 2 e_z of itself; gradients' entries by 3 e_z of the sum of the sizes of their terms, plus half a step of
            their type
"""
import math

import pytest
import torch

from test_hip_vocab import DT, HALF, U, _inputs, _leaves, _run_ce, _teacher


def _e_z(K, z):
    return 8 * K ** 0.5 * U * (float(z[torch.isfinite(z)].abs().max()) + 1)


def _exact(h, w, b, ids, p, T, g):
    """Losses and gradients in 64 bits, by the formulas; ids / p (R, S), g (R,).  Also the sums of the sizes of the gradients' terms."""
    H, W = h.double(), w.double()
    z = H @ W.t()
    if b is not None:
        z = z + b.double()
    z = z / T
    L = torch.logsumexp(z, 1)
    zt = z.gather(1, ids)
    logp = torch.where(p > 0, p.log(), torch.zeros_like(p))
    loss = T * T * (p * (logp - torch.where(p > 0, zt, torch.zeros_like(zt)) + L[:, None])).sum(1)
    q = (z - L[:, None]).exp()
    target = torch.zeros_like(q).scatter_add_(1, ids, p)
    gt = (g.double() * T)[:, None]
    dS, size = gt * (q - target), gt.abs() * (q + target)
    out = {"loss": loss, "d_hidden": dS @ W, "d_weight": dS.t() @ H, "d_bias": dS.sum(0)}
    sizes = {"d_hidden": size @ W.abs(), "d_weight": size.t() @ H.abs(), "d_bias": size.sum(0)}
    return z, out, sizes


# ---- the gradient of the scores is not what 16-bit gradients show ----
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("R,V,K", [(300, 5003, 512), (1030, 5003, 264), (3000, 9001, 256)])
@pytest.mark.parametrize("loss", ["cross_entropy", "distillation"])
def test_gradients_of_many_16_bit_rows_are_rounded_once(dtype, R, V, K, loss):
    """The error of a 16-bit gradient is that of its own rounding.  dS in two 16-bit planes is off by at most half a step squared of an
    entry (2^-16, 2^-22); against the half step of the result that is 2^-8 at most, and the squares of independent errors add: (1 + 2^-16)
    under the root; sums of K or R fp32 terms are far below.  1.02 leaves room for few entries (d_bias: V of them).  One plane of dS gives 1.4."""
    from gridmm_amd import vocab
    h, w, b, g = _inputs(dtype, R, V, K, True, seed=R)
    gr = (torch.rand(R, generator=g) + 0.5).cuda()
    hl, wl, bl = _leaves(h, w, b)
    if loss == "cross_entropy":
        ids = torch.randint(0, V, (R, 1), generator=g).cuda()
        p, T = torch.ones(R, 1, dtype=torch.float64, device="cuda"), 1.0
        vocab.vocab_cross_entropy(hl, wl, ids[:, 0], bias=bl).backward(gr)
    else:
        T = 2.0
        ids = torch.stack([torch.randperm(V, generator=g)[:16] for _ in range(R)]).cuda()
        t = (torch.randn(R, 16, generator=g) * 3).cuda()
        p = _teacher(ids, t, T)
        vocab.vocab_distillation(hl, wl, ids, t, bias=bl, temperature=T).backward(gr)
    _, want, _ = _exact(h, w, b, ids, p, T, gr)
    for k, x in (("d_hidden", hl.grad), ("d_weight", wl.grad), ("d_bias", bl.grad)):
        own = want[k].to(DT[dtype]).double() - want[k]
        ratio = float((x.double() - want[k]).norm() / own.norm())
        assert ratio <= 1.02, (k, ratio)


# ---- rows that the model is sure of ----
def _sure(dtype, R, V, K, margin, seed):
    """Hidden states that lie along the row of W of their label: the label's score is `margin` above everything else's typical one."""
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(V, K, generator=g) / K ** 0.5
    y = torch.randperm(V, generator=g)[:R]
    h = w[y] * (margin / (w[y] * w[y]).sum(1, keepdim=True)) + 0.1 * torch.randn(R, K, generator=g)
    return h.to(DT[dtype]).cuda(), w.to(DT[dtype]).cuda(), y.cuda(), g


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("R,V,K", [(20, 700, 256), (300, 4000, 768), (400, 30011, 260), (2600, 11000, 256)])
@pytest.mark.parametrize("margin", [14.0, 34.0])
@pytest.mark.parametrize("loss", ["cross_entropy", "one slot", "three slots"])
def test_rows_that_the_model_is_sure_of(dtype, R, V, K, margin, loss):
    """loss = (M - z_y) + log sum 2^(y - M): where the label's score is the maximum M the first term is 0 if both come from one product,
    and the second one is a sum that starts at 1: at most 64 additions next to 1 (a lane's columns, the lanes, the tiles), each off by
    u, exponentials off by 3 e_z of themselves, a logarithm off by 4 u: never below 0.  The label's entry of dS is
    g (1 / sum - 1) likewise."""
    from gridmm_amd import vocab
    h, w, y, g = _sure(dtype, R, V, K, margin, seed=V)
    # distinct powers of two: d_bias of a label is its row's entry of dS plus what other rows leave there
    gr = torch.ones(R, device="cuda")
    b = torch.zeros(V, dtype=torch.float32, device="cuda")
    hl, wl, bl = _leaves(h, w, b)
    if loss == "cross_entropy":
        ids, p = y[:, None], torch.ones(R, 1, dtype=torch.float64, device="cuda")
        got = vocab.vocab_cross_entropy(hl, wl, y, bias=bl)
    else:
        S = 1 if loss == "one slot" else 3
        ids = torch.stack([y] + [(y + 1 + s) % V for s in range(S - 1)], 1)
        t = torch.full((R, S), -200.0, device="cuda")      # (the others' share: e^-300, nothing in fp32)
        t[:, 0] = 100.0
        p = torch.zeros(R, S, dtype=torch.float64, device="cuda")
        p[:, 0] = 1.0
        got = vocab.vocab_distillation(hl, wl, ids, t, bias=bl)
    got.backward(gr)
    z, want, _ = _exact(h, w, b, ids, p, 1.0, gr)
    ez = _e_z(K, z)
    bound = want["loss"] * 3 * ez + 68 * U
    sure = z.gather(1, y[:, None])[:, 0] == z.max(1)[0]
    assert int(sure.sum()) > 0.9 * R
    got = got.detach().double()
    assert bool((got[sure] >= 0).all()), float(got[sure].min())
    err = ((got - want["loss"]).abs() - bound)[sure]
    assert float(err.max()) <= 0, (float(err.max()), float(bound.max()))
    # d_bias[y_r] = (q - 1) + the q of the other rows there: the entry, rounded to two 16-bit planes, and a sum of R terms
    e = (1 - want["loss"].neg().exp()) * (3 * ez + 2.0 ** -16) + 68 * U
    q = (z - torch.logsumexp(z, 1, keepdim=True)).exp().sum(0)[y] - want["loss"].neg().exp()
    d = (bl.grad.double()[y] - want["d_bias"][y]).abs() - e - q.abs() * (3 * ez + 2.0 ** -16 + R * U) - R * 2.0 ** -38
    assert float(d[sure].max()) <= 0, float(d[sure].max())


# ---- rows of very different size ----
def _neighbours(got, want, sizes, z, h, rows, columns, dtype):
    """Losses and gradients of `rows`, and the gradients of `columns` of the vocabulary, to what fp32 products leave."""
    K, half = h.shape[1], HALF[DT[dtype]]
    ez = _e_z(K, z[rows])
    assert float(((got["loss"].double() - want["loss"]).abs()[rows]).max()) <= 3 * ez + 8 * U * float(want["loss"][rows].abs().max())
    for k, at in (("d_hidden", rows), ("d_weight", columns), ("d_bias", columns)):
        v, n = want[k][at], sizes[k][at]
        d = (got[k].double()[at] - v).abs() - 3 * ez * n - half * v.abs()
        if dtype == "fp16":
            d = d - 2.0 ** -25
        assert float(d.max()) <= 0, (k, float(d.max()), float(n.max()))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("R,V,K", [(20, 500, 64), (300, 4000, 768), (500, 30011, 100), (2600, 11000, 96)])
@pytest.mark.parametrize("factor", [1e4, 1e8, 1e12, 1e30])
def test_one_large_hidden_row_leaves_the_others_alone(dtype, R, V, K, factor):
    h, w, b, g = _inputs(dtype, R, V, K, True, seed=3)
    h[5] *= factor
    labels = torch.randint(0, V, (R,), generator=g).cuda()
    gr = (torch.rand(R, generator=g) + 0.5).cuda()
    got = _run_ce(h, w, b, labels, gr)
    z, want, sizes = _exact(h, w, b, labels[:, None], torch.ones(R, 1, dtype=torch.float64, device="cuda"), 1.0, gr)
    rows = torch.arange(R, device="cuda") != 5
    columns = torch.ones(V, dtype=torch.bool, device="cuda")
    columns[labels[5]] = False                     # the large row reaches these two
    columns[z[5].argmax()] = False
    _neighbours(got, want, sizes, z, h, rows, columns, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("R,V,K", [(20, 500, 64), (300, 4000, 768), (500, 30011, 100), (2600, 11000, 96)])
@pytest.mark.parametrize("factor", [1e4, 1e8, 1e12, 1e30])
@pytest.mark.parametrize("masked", [True, False])
def test_one_large_row_of_the_weight_leaves_the_others_alone(dtype, R, V, K, factor, masked):
    """A column masked by its bias; or one whose large scores are negative for half of the rows, which keep theirs."""
    h, w, b, g = _inputs(dtype, R, V, K, True, seed=4)
    w[7] *= factor
    if masked:
        b[7] = float("-inf")
    labels = torch.randint(8, V, (R,), generator=g).cuda()
    gr = (torch.rand(R, generator=g) + 0.5).cuda()
    z7 = h.double() @ w[7].double()
    rows = torch.ones(R, dtype=torch.bool, device="cuda") if masked else z7 < -200
    gr = torch.where(rows, gr, torch.zeros_like(gr))
    got = _run_ce(h, w, b, labels, gr)
    keep = torch.arange(V, device="cuda") != 7
    z, want, sizes = _exact(h, w[keep], b[keep], (labels - 1)[:, None], torch.ones(R, 1, dtype=torch.float64, device="cuda"), 1.0, gr)
    assert int(rows.sum()) > R // 8
    got["d_weight"], got["d_bias"], seven = got["d_weight"][keep], got["d_bias"][keep], got["d_weight"][7]
    _neighbours(got, want, sizes, z, h, rows, torch.ones(V - 1, dtype=torch.bool, device="cuda"), dtype)
    assert bool((seven == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("S", [3, 90])
def test_distillation_beside_one_large_row(S):
    from gridmm_amd import vocab
    R, V, K, T = 600, 3000, 1000, 2.0
    h, w, b, g = _inputs("fp32", R, V, K, True, seed=6)
    h[5] *= 1e10
    w[7] *= 1e10
    b[7] = float("-inf")
    ids = torch.stack([8 + torch.randperm(V - 8, generator=g)[:S] for _ in range(R)]).cuda()
    t = torch.randn(R, S, generator=g).cuda()
    gr = (torch.rand(R, generator=g) + 0.5).cuda()
    hl, wl, bl = _leaves(h, w, b)
    loss = vocab.vocab_distillation(hl, wl, ids, t, bias=bl, temperature=T)
    loss.backward(gr)
    keep = torch.arange(V, device="cuda") != 7
    z, want, sizes = _exact(h, w[keep], b[keep], ids - 1, _teacher(ids, t, T), T, gr)
    got = {"loss": loss.detach() / (T * T), "d_hidden": hl.grad, "d_weight": wl.grad[keep], "d_bias": bl.grad[keep]}
    want["loss"] = want["loss"] / (T * T)
    columns = torch.ones(V - 1, dtype=torch.bool, device="cuda")
    columns[ids[5] - 1] = False
    columns[z[5].argmax()] = False
    _neighbours(got, want, sizes, z, h, torch.arange(R, device="cuda") != 5, columns, "fp32")


@pytest.mark.gpu
@pytest.mark.parametrize("loss", ["cross_entropy", "distillation"])
@pytest.mark.parametrize("dtype,R,V,K", [("fp32", 9100, 33001, 72), ("fp16", 9100, 33001, 72), ("fp32", 270, 200003, 700)])
def test_rows_far_apart_over_several_pieces(dtype, R, V, K, loss):
    """More columns than a piece of dS or a packed piece of W holds, rows of wider matrices off 16-byte boundaries, ignored rows among them: an
    outlier row of each operand (fp32), upstream gradients far apart."""
    from gridmm_amd import vocab
    h, w, b, g = _inputs(dtype, R, V, K, True, seed=7)
    if dtype == "fp32":
        h[5] *= 1e9
        w[7] *= 1e9
    b[7] = float("-inf")

    def strided(t):
        return torch.zeros(t.shape[0], t.shape[1] + 5, dtype=t.dtype, device="cuda")[:, 3:3 + t.shape[1]].copy_(t)
    hl, wl, bl = _leaves(strided(h), strided(w), b)
    gr = (torch.rand(R, generator=g) + 0.5).cuda()
    gr[::3] *= 2.0 ** -24
    if dtype == "fp16":
        gr *= 2.0 ** 12
    live = torch.rand(R, generator=g).cuda() > 0.2
    live[5] = True
    S, T = (1, 1.0) if loss == "cross_entropy" else (4, 2.0)
    ids = (8 + torch.stack([torch.randperm(V - 8, generator=g)[:S] for _ in range(R)])).cuda()
    p = torch.ones(R, S, dtype=torch.float64, device="cuda")
    if loss == "cross_entropy":
        got = vocab.vocab_cross_entropy(hl, wl, torch.where(live, ids[:, 0], torch.full_like(ids[:, 0], -1)), bias=bl)
    else:
        t = torch.randn(R, S, generator=g).cuda()
        p = _teacher(ids, t, T)
        got = vocab.vocab_distillation(hl, wl, torch.where(live[:, None], ids, torch.full_like(ids, -1)), t, bias=bl, temperature=T)
    got.backward(gr)
    keep = torch.arange(V, device="cuda") != 7
    z, want, sizes = _exact(h, w[keep], b[keep], ids - 1, p, T, torch.where(live, gr, torch.zeros_like(gr)))
    want["loss"] = torch.where(live, want["loss"], torch.zeros_like(want["loss"])) / (T * T)
    rows = torch.arange(R, device="cuda") != 5 if dtype == "fp32" else torch.ones(R, dtype=torch.bool, device="cuda")
    columns = torch.ones(V - 1, dtype=torch.bool, device="cuda")
    if dtype == "fp32":
        columns[ids[5] - 1] = False
        columns[z[5].argmax()] = False
    out = {"loss": got.detach() / (T * T), "d_hidden": hl.grad, "d_weight": wl.grad[keep], "d_bias": bl.grad[keep]}
    z[~live] = 0.0
    _neighbours(out, want, sizes, z, h, rows, columns, dtype)
    assert bool((hl.grad[~live] == 0).all()) and bool((wl.grad[7] == 0).all())


# ---- upstream gradients far apart ----
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("R,V,K", [(30, 20000, 64), (300, 30011, 96), (2600, 11000, 96)])
@pytest.mark.parametrize("ratio", [10, 18, 30])
def test_rows_of_small_upstream_gradients_keep_their_own(dtype, R, V, K, ratio):
    """Nearly flat rows against a weight with a mean of its own: the many small entries of dS make up as much of dh as the label's.  Rows
    whose upstream gradient is 2^-ratio of the others' are held to their own size."""
    h, w, b, g = _inputs(dtype, R, V, K, True, seed=2, spread=0.3)
    w = (w.float() + torch.randn(K, generator=g).cuda()).to(DT[dtype])
    h = (h.float() * 0.05).to(DT[dtype])
    labels = torch.randint(0, V, (R,), generator=g).cuda()
    gr = (torch.rand(R, generator=g) + 0.5).cuda()
    gr[::2] *= 2.0 ** -ratio
    if dtype == "fp16":
        gr *= 2.0 ** min(ratio, 14)                # (dh itself has fp16's range)
    got = _run_ce(h, w, b, labels, gr)
    z, want, sizes = _exact(h, w, b, labels[:, None], torch.ones(R, 1, dtype=torch.float64, device="cuda"), 1.0, gr)
    every = torch.ones(R, dtype=torch.bool, device="cuda")
    _neighbours(got, want, sizes, z, h, every, torch.ones(V, dtype=torch.bool, device="cuda"), dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("R,V,K,apart", [(300, 4000, 768, 32), (300, 4000, 768, 17), (2600, 11000, 256, 32)])
def test_columns_that_only_rows_of_small_gradients_reach(dtype, R, V, K, apart):
    """Rows that put everything on one column, their label another: the label's entry of dS is -g, the column's +g.  The rows of the even half
    have upstream gradients 2^-apart of the others' and hidden states up to 2^12 times as large (another bias holds their scores down), so that the
    columns that only they reach have sums of their own size."""
    g = torch.Generator().manual_seed(apart)
    w = torch.randn(V, K, generator=g) / K ** 0.5
    order = torch.randperm(V, generator=g)[:2 * R]
    top, labels = order[:R], order[R:2 * R].cuda()
    h = w[top] * (40.0 / (w[top] * w[top]).sum(1, keepdim=True))
    up = 12 if apart == 32 else 0
    h[::2] *= 2.0 ** up
    h, w = h.to(DT[dtype]).cuda(), w.to(DT[dtype]).cuda()
    gr = (torch.rand(R, generator=g) + 0.5).cuda()
    gr[::2] *= 2.0 ** -apart
    b = torch.zeros(V, device="cuda")
    hl, wl, bl = _leaves(h, w, b)
    from gridmm_amd import vocab
    vocab.vocab_cross_entropy(hl, wl, labels, bias=bl).backward(gr * 2.0 ** 14 if dtype == "fp16" else gr)
    gx = gr * 2.0 ** 14 if dtype == "fp16" else gr
    z, want, sizes = _exact(h, w, b, labels[:, None], torch.ones(R, 1, dtype=torch.float64, device="cuda"), 1.0, gx)
    half = HALF[DT[dtype]]
    # a row's other entries of dS: softmax of scores 40 apart at least less what 8 standard deviations make up; far below fp32 where h is larger
    for k, got in (("d_bias", bl.grad), ("d_weight", wl.grad)):
        at = labels[::2]
        v = want[k][at]
        # the entry itself: (1 - q) g, two 16-bit planes (2^-16).  The layout of h has rows' |g h| up to 2^20 apart, the largest in [2^14, 2^15): a row's
        # largest value lies at 2^-6 at least, and half of fp16's last step is 2^-25, so a value is off by 2^-19 of its row's largest at most
        bound = (2.0 ** -15 + (half if k == "d_weight" else 0.0)) * sizes[k][at] + (2.0 ** -25 if dtype == "fp16" else 0.0)
        if k == "d_weight":
            bound = bound + 2.0 ** -19 * (gx[::2].double() * h[::2].double().abs().amax(1))[:, None]
        d = (got.double()[at] - v).abs() - bound
        assert float(d.max()) <= 0, (k, float(d.max()), float(v.abs().max()))
        assert float(v.abs().max()) > 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "fp16"])
def test_a_captured_step_finds_out_anew_at_each_replay(dtype):
    """Whether one scale serves all rows is decided on the device: a graph captured with ordinary rows is replayed with an outlier, with
    upstream gradients far apart, and with ordinary ones again; every replay equals the eager call."""
    from gridmm_amd import vocab
    R, V, K = 300, 20011, 192
    h, w, b, g = _inputs(dtype, R, V, K, True, seed=8)
    hl, wl, bl = _leaves(h, w, b)
    labels = torch.randint(0, V, (R,), generator=g).cuda()
    gr = (torch.rand(R, generator=g) + 0.5).cuda()
    plain = gr.clone()

    def step():
        loss = vocab.vocab_cross_entropy(hl, wl, labels, bias=bl)
        return (loss,) + torch.autograd.grad(loss, (hl, wl, bl), gr)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        step()
    torch.cuda.current_stream().wait_stream(st)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for large, ratio in ((1.0, 0), (3e4, 0), (1.0, 30), (1.0, 0), (3e4, 30)):
        with torch.no_grad():
            hl.copy_(h)
            hl[7] *= large
        gr.copy_(plain)
        gr[::3] *= 2.0 ** -ratio
        graph.replay()
        torch.cuda.synchronize()
        want = _run_ce(hl.detach(), w, b, labels, gr)
        for x, k in zip(out, ("loss", "d_hidden", "d_weight", "d_bias")):
            assert torch.equal(torch.nan_to_num(x), torch.nan_to_num(want[k])), (large, ratio, k)


# ---- no tile is left out ----
@pytest.mark.gpu
@pytest.mark.parametrize("dtype,R,V,K", [("bf16", 300, 70000, 64), ("fp32", 300, 70000, 64), ("fp16", 300, 33000, 72), ("fp32", 20, 9001, 64),
                                         ("bf16", 9100, 33001, 72), ("fp32", 2100, 40003, 128), ("fp32", 270, 300001, 520)])
def test_every_tile_counts(dtype, R, V, K):
    """Each block of 64 columns in turn holds the column that makes up nearly all of a row's sum, and each in turn the label: a block left
    out of the sum, the scores or the gradients changes a loss by more than 5.  Then flat rows: the sum of V equal terms is off by less
    than half of what one block of 64 columns is of it."""
    from gridmm_amd import vocab
    g = torch.Generator().manual_seed(V)
    w = torch.randn(V, K, generator=g)
    w = (w * (4.0 / w.norm(dim=1, keepdim=True))).to(DT[dtype])
    blocks = (V + 63) // 64
    at = torch.arange(max(R, blocks)) % blocks
    top = (at * 64 + torch.randint(0, 64, at.shape, generator=g)).clamp(max=V - 1)
    label = ((at * 7919 + 13) % blocks * 64 + torch.randint(0, 64, at.shape, generator=g)).clamp(max=V - 1)
    w, label, top = w.cuda(), label.cuda(), top.cuda()
    for r0 in range(0, at.numel(), R):
        t, y = top[r0:r0 + R], label[r0:r0 + R]
        h = (w[t].float() * (24.0 / 16.0)).to(DT[dtype])
        hl = h.requires_grad_()
        loss = vocab.vocab_cross_entropy(hl, w, y)
        z = h.detach().double() @ w.double().t()
        L = torch.logsumexp(z, 1)
        want = L - z.gather(1, y[:, None])[:, 0]
        ez = _e_z(K, z)
        near = (loss.detach().double() - want).abs() <= 3 * ez + 8 * U * 40
        assert bool(near.all()), (r0, int((~near).sum()))
        if r0 == 0:
            assert float((L - torch.logsumexp(z.scatter(1, t[:, None], float("-inf")), 1)).min()) > 5
        loss.sum().backward()
        dS = (z - L[:, None]).exp()
        dS.scatter_add_(1, y[:, None], torch.full_like(y[:, None], -1, dtype=torch.float64))
        d = hl.grad.double() - dS @ w.double()
        assert float(d.abs().max()) <= (3 * ez * 2 + HALF[DT[dtype]] * 2) * 4, r0
        del z, dS, d, hl, loss
    flat = (torch.randn(min(R, 300), K, generator=g) * 2.0 ** -12).to(DT[dtype]).cuda()
    y = label[:flat.shape[0]]
    loss = vocab.vocab_cross_entropy(flat, w, y).double()
    z = flat.double() @ w.double().t()
    bound = 3 * _e_z(K, z) + 8 * U * math.log(V)
    assert bound < 32.0 / V
    assert float((loss - torch.logsumexp(z, 1) + z.gather(1, y[:, None])[:, 0]).abs().max()) <= bound


# ---- no rows ----
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_no_rows_under_a_frozen_decoder(dtype):
    """A batch without a masked token whose decoder is not trained: an empty gradient, not an error."""
    from gridmm_amd import vocab
    h, w, b, _ = _inputs(dtype, 0, 100, 64)
    hl = h.requires_grad_()
    vocab.vocab_cross_entropy(hl, w, torch.zeros(0, dtype=torch.long, device="cuda"), bias=b).sum().backward()
    assert hl.grad.shape == (0, 64)
    hl.grad = None
    vocab.vocab_distillation(hl, w, torch.zeros(0, 3, dtype=torch.long, device="cuda"), torch.zeros(0, 3, device="cuda"), bias=b).sum().backward()
    assert hl.grad.shape == (0, 64)


def test_no_rows_and_no_outputs_at_the_c_entry():
    """Nothing is launched: an empty hidden gradient has no address."""
    import ctypes
    from test_hip_vocab import _descriptor
    from gridmm_amd import _lib
    lib = _lib.load()
    d = _descriptor(rows=0, weight=256)
    assert lib.gridmm_vocab_loss_bwd(ctypes.byref(d), 256, 1 << 40, None, 1, None, None, None, 256, 1 << 40, None) == 0


# ---- memory ----
@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("rows", [1000, 16384, 40000, 2 ** 17, 2 ** 20])
@pytest.mark.parametrize("vocab,hidden", [(30522, 768), (131072, 2048), (131072, 33001), (5000, 64), (2 ** 17, 2 ** 20)])
def test_workspaces_stay_within_what_is_said_of_them(dtype, rows, vocab, hidden):
    """The library is asked without a GPU."""
    import ctypes
    from test_hip_vocab import _descriptor
    from gridmm_amd import _lib
    lib = _lib.load()
    d = _descriptor(rows=rows, vocab=vocab, hidden_size=hidden, dtype=dtype, bias_dtype=dtype, ld_hidden=hidden, ld_weight=hidden, hidden=256, weight=256)
    size, MB = 4 if dtype == 0 else 2, 2 ** 20
    rp, vp, kp = (rows + 255) // 256 * 256, (vocab + 255) // 256 * 256, (hidden + 63) // 64 * 64
    piece_w = max(512 * MB, 256 * kp * size)
    saved = lib.gridmm_vocab_loss_saved_bytes(ctypes.byref(d))
    assert 0 < saved <= rp * kp * size + 512 * MB + 64 * rp + 4 * vp + 4096
    forward = lib.gridmm_vocab_loss_workspace(ctypes.byref(d), 0)
    assert 0 < forward <= rp * vp // 16 + piece_w + 64 * rp + 65536
    backward = lib.gridmm_vocab_loss_workspace(ctypes.byref(d), 1)
    scores_grad, sums, layout = max(512 * MB, 32768 * rp), max(256 * MB, 4 * rp * kp), 0 if dtype == 1 else rp * kp * size
    assert 0 < backward <= scores_grad + sums + layout + piece_w + 64 * rp + 65536


# ---- extreme values: top logits ----
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("R,V", [(1, 70001), (3, 300), (300, 9001), (2000, 3000)])
def test_top_logits_of_rows_masked_with_large_finite_numbers(dtype, R, V):
    """Masks of -1e9 to -1e38 and the lowest number, in whole stretches and here and there, and rows whose own values are that large: the
    log-sum-exp is that of the rest, sums of V exponentials (sqrt(V) + 16) u off, or as large as the largest value."""
    from gridmm_amd import vocab
    g = torch.Generator().manual_seed(V)
    for mask in (-1e9, -3e10, -1e20, -1e30, -9e37, float(torch.finfo(DT[dtype]).min)):
        x = torch.randn(R, V, generator=g) * 3
        x[:, : V // 2] = mask
        x[torch.rand(R, V, generator=g) < 0.3] = mask
        x[:, -1] = 1.0
        x = x.to(DT[dtype]).cuda()
        values, ids, lse = vocab.top_logits(x, 5)
        want, order = x.float().sort(dim=1, descending=True, stable=True)
        assert torch.equal(ids, order[:, :5]) and torch.equal(values.float(), want[:, :5])
        z = torch.logsumexp(x.double(), 1)
        assert float((lse.double() - z).abs().max()) <= (V ** 0.5 + 16) * U * 30, mask
    for size in (1e9, 3e10, 1e20, 1e37, 2e38):
        x = (torch.randn(R, V, generator=g) * size / 8).to(DT[dtype]).cuda()
        lse = vocab.top_logits(x, 1)[2].double()
        z = torch.logsumexp(x.double(), 1)
        # (2e38: rows that hold an infinity have it as their log-sum-exp, exactly)
        off = torch.where(lse == z, torch.zeros_like(z), (lse - z).abs() / z.abs())
        assert float(off.max()) <= 4 * U, size


# ---- extreme values: teachers ----
@pytest.mark.gpu
@pytest.mark.parametrize("R,V,K", [(10, 300, 64), (300, 4000, 768)])
@pytest.mark.parametrize("T", [0.25, 1.0, 4.0])
def test_a_teacher_with_extreme_values(R, V, K, T):
    """Slots masked with the lowest number, rows of nothing else, and logits whose quotient by T is no longer a number of fp32."""
    from gridmm_amd import vocab
    h, w, b, g = _inputs("fp32", R, V, K, True, seed=1)
    ids = torch.stack([torch.randperm(V, generator=g)[:6] for _ in range(R)]).cuda()
    t = torch.randn(R, 6, generator=g).cuda()
    low = torch.finfo(torch.float32).min
    t[0, 2:] = low                                 # two slots count
    t[1] = low                                     # all alike
    t[2] = 3e38
    t[3, 1:] = -3e38
    t[4, 0] = 3e38                                 # one slot has it all
    hl = h.clone().requires_grad_()
    gr = torch.ones(R, device="cuda")
    loss = vocab.vocab_distillation(hl, w, ids, t, bias=b, temperature=T)
    loss.backward(gr)
    z, want, sizes = _exact(h, w, b, ids, _teacher(ids, t, T), T, gr)
    ez = _e_z(K, z)
    assert float((loss.detach().double() - want["loss"]).abs().max()) <= T * T * (3 * ez + 16 * U * 8)
    assert float(((hl.grad.double() - want["d_hidden"]).abs() - 3 * ez * sizes["d_hidden"]).max()) <= 0


# ---- extreme values: nothing left ----
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("R,V,K", [(10, 300, 64), (300, 4000, 768)])
@pytest.mark.parametrize("mask", ["-inf", "lowest"])
def test_rows_without_a_column_are_no_number(dtype, R, V, K, mask):
    """All columns out of the softmax: 0 / 0."""
    from gridmm_amd import vocab
    h, w, b, g = _inputs(dtype, R, V, K, True, seed=1)
    b[:] = float("-inf") if mask == "-inf" else torch.finfo(b.dtype).min
    y = torch.randint(0, V, (R,), generator=g).cuda()
    y[1] = -1
    hl = h.requires_grad_()
    for loss in (vocab.vocab_cross_entropy(hl, w, y, bias=b),
                 vocab.vocab_distillation(hl, w, torch.stack([y, y], 1), torch.zeros(R, 2, device="cuda"), bias=b)):
        assert float(loss[1]) == 0.0
        rest = torch.arange(R, device="cuda") != 1
        assert bool(torch.isnan(loss[rest]).all())
        d, = torch.autograd.grad(loss.sum(), hl)
        assert bool(torch.isnan(d[rest]).all()) and bool((d[1] == 0).all())
