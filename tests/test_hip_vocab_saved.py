"""The vocabulary losses under saved-tensor hooks: checkpointing and offloading give the backward other tensors than the forward had, whose
memory may be in use for something else by then.  The kernels have to read the ones that come back."""
import contextlib
import ctypes

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from test_hip_vocab import DT, _inputs


class _Library:
    """Stands for the library: notes the descriptors of the calls, and what its addresses point to."""

    def __init__(self):
        self.forward, self.backward = [], []

    def gridmm_vocab_loss_saved_bytes(self, d):
        return 256

    def gridmm_vocab_loss_workspace(self, d, backward):
        return 256

    @staticmethod
    def _note(d, index_bytes=8):
        d = d._obj
        one = lambda p, n: None if not p else ctypes.string_at(p, n)
        return dict(hidden=d.hidden, weight=d.weight, bias=d.bias, index=d.ids if d.slots else d.labels, ld=(d.ld_hidden, d.ld_weight, d.ld_ids),
                    first=[one(p, 4) for p in (d.hidden, d.weight, d.bias)] + [one(d.ids if d.slots else d.labels, index_bytes)])

    def gridmm_vocab_loss_fwd(self, d, *args):
        self.forward.append(self._note(d))
        return 0

    def gridmm_vocab_loss_bwd(self, d, *args):
        self.backward.append(self._note(d))
        return 0


@pytest.fixture
def library(monkeypatch):
    from gridmm_amd import _lib, vocab
    lib = _Library()
    monkeypatch.setattr(_lib, "load", lambda *a, **k: lib)
    monkeypatch.setattr(vocab, "_on", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(vocab, "_stream", lambda: None)
    return lib


def _call(h, w, b, index, t=None):
    from gridmm_amd import vocab
    return vocab._VocabLoss.apply(h, w, b, index, t, -1, 1.0, torch.is_grad_enabled())


def _cpu_inputs(slots):
    g = torch.Generator().manual_seed(0)
    x = torch.randn(6, 16, generator=g, requires_grad=True)
    w = torch.randn(10, 16, generator=g, requires_grad=True)
    b = torch.randn(10, generator=g, requires_grad=True)
    if slots:
        return x, w, b, torch.arange(30).view(6, 5)[:, 1:4] % 10, torch.randn(6, 3, generator=g)
    return x, w, b, torch.arange(6), None


@pytest.mark.parametrize("slots", [False, True])
def test_a_checkpointed_backward_reads_what_the_second_forward_kept(library, slots):
    x, w, b, index, t = _cpu_inputs(slots)
    keep = []

    def head(x):
        keep.extend(torch.empty_like(x) for _ in range(256))      # (the memory of the first forward's h is taken: the second's lies elsewhere)
        return _call(x * 2.0, w, b, index, t)
    checkpoint(head, x, use_reentrant=False).sum().backward()
    assert len(library.forward) == 2 and len(library.backward) == 1
    first, second, back = library.forward[0], library.forward[1], library.backward[0]
    assert first["hidden"] != second["hidden"] and back["hidden"] == second["hidden"]
    assert back["first"] == second["first"]


@pytest.mark.parametrize("slots", [False, True])
def test_the_backward_reads_the_tensors_that_the_hooks_give_back(library, slots):
    """Copies, in another layout for the ids, while the originals are overwritten by the next user of their memory."""
    x, w, b, index, t = _cpu_inputs(slots)
    given = []

    def unpack(t):
        given.append(t.clone())
        return given[-1]
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), unpack):
        loss = _call(x * 2.0, w, b, index, t)
    loss.sum().backward()
    back, there = library.backward[0], {t.data_ptr(): t for t in given}
    for k in ("hidden", "weight", "bias", "index"):
        assert back[k] in there, k
    ld = (16, 16, there[back["index"]].stride(0) if slots else 0)
    assert back["ld"] == ld
    assert back["first"] == library.forward[0]["first"]


def test_a_tensor_that_comes_back_as_something_else_is_refused(library):
    for change in (lambda t: t.double() if t.dtype == torch.float32 else t, lambda t: t[:-1] if t.dtype == torch.float32 else t):
        x, w, b, index, t = _cpu_inputs(False)
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change):
            loss = _call(x * 2.0, w, b, index)
        with pytest.raises(RuntimeError, match="other shapes or types"):
            loss.sum().backward()
    assert not library.backward


def test_nothing_but_parameters_is_kept_beside_the_saved_tensors(library):
    import weakref
    x, w, b, index, _ = _cpu_inputs(False)
    cast = w * 1.0
    gone = weakref.ref(cast)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), lambda t: t):
        loss = _call(x, cast, b, index)
    node = loss.grad_fn
    assert not any(t is cast for t in node.prm) and node.prm == [None, None]
    del cast, node
    assert gone() is None


# ---- on the GPU ----
def _grads(f, leaves):
    loss = f()
    return (loss.detach(),) + torch.autograd.grad(loss, leaves, torch.linspace(0.5, 1.5, loss.numel(), device="cuda"))


def _overwrite():
    """Whatever memory is free gets other contents."""
    for n in (1 << 12, 1 << 16, 1 << 20, 1 << 24):
        for _ in range(4):
            torch.full((n,), float("nan"), device="cuda")


SIZES = [("fp32", 9, 700, 64), ("bf16", 9, 700, 72), ("fp32", 300, 20011, 192), ("bf16", 300, 20011, 192), ("fp16", 300, 20011, 200)]


def _heads(dtype, R, V, K):
    """Both losses as functions of an intermediate hidden state, with temporaries behind every argument."""
    from gridmm_amd import vocab
    h, w, b, g = _inputs(dtype, R, V, K, True, seed=V)
    x, wt, b = h.requires_grad_(), w.t().contiguous().requires_grad_(), b.requires_grad_()
    labels = torch.randint(0, V, (R, 2), generator=g).cuda()
    table = torch.randint(0, V, (R, 9), generator=g).cuda()
    t = torch.randn(R, 9, generator=g).cuda()

    def ce(x):
        return vocab.vocab_cross_entropy(x * 1.5, wt.t(), labels[:, 1] + 0, bias=b + 0)

    def kd(x):
        return vocab.vocab_distillation(x * 1.5, wt.t(), (table + 0)[:, 2:7], t[:, 1:6] * 2, bias=b + 0, temperature=2.0)
    return x, wt, b, ce, kd


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,R,V,K", SIZES)
def test_under_checkpointing(dtype, R, V, K):
    x, wt, b, ce, kd = _heads(dtype, R, V, K)

    def checked(f):
        def g(x):
            loss = checkpoint(f, x, use_reentrant=False)
            _overwrite()
            return loss
        return g
    for f in (ce, kd):
        want = _grads(lambda: f(x), (x, wt, b))
        got = _grads(lambda: checked(f)(x), (x, wt, b))
        for a, c in zip(want, got):
            assert torch.equal(a, c)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,R,V,K", SIZES)
@pytest.mark.parametrize("how", ["offload", "copies", "unaligned"])
def test_under_saved_tensor_hooks(dtype, R, V, K, how):
    """Offloaded to the host and back; copies on the device; copies off every 16-byte boundary in rows of another stride."""
    x, wt, b, ce, kd = _heads(dtype, R, V, K)

    def unaligned(t):
        if t.dim() < 2 or t.dtype == torch.uint8:
            return t.clone()
        out = torch.empty(t.shape[0], t.shape[1] + 3, dtype=t.dtype, device=t.device)[:, 1:1 + t.shape[1]]
        return out.copy_(t)
    hooks = {"offload": lambda: torch.autograd.graph.save_on_cpu(), "unaligned": lambda: torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), unaligned),
             "copies": lambda: torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), lambda t: t.clone())}[how]
    for f in (ce, kd):
        def hooked():
            with hooks():
                loss = f(x)
            _overwrite()
            return loss
        want = _grads(lambda: f(x), (x, wt, b))
        got = _grads(hooked, (x, wt, b))
        for a, c in zip(want, got):
            if how == "unaligned" and R < 20:      # (few rows: loads of another width, sums in another order)
                assert float((a.double() - c.double()).abs().max()) <= 2.0 ** -7 * float(a.double().abs().max())
            else:
                assert torch.equal(a, c)


@pytest.mark.gpu
@pytest.mark.parametrize("R,V,K", [(9, 700, 64), (300, 20011, 192)])
def test_a_parameter_whose_storage_was_exchanged(R, V, K):
    """The forward's storage is gone; the backward takes the values that the parameter has now, as torch's own nodes do."""
    from gridmm_amd import vocab
    h, w, b, g = _inputs("bf16", R, V, K, True, seed=V)
    labels = torch.randint(0, V, (R,), generator=g).cuda()
    p = torch.nn.Parameter(w.clone())
    x = h.requires_grad_()
    want = torch.autograd.grad(vocab.vocab_cross_entropy(x, p, labels, bias=b).sum(), (x, p))
    loss = vocab.vocab_cross_entropy(x, p, labels, bias=b).sum()
    p.data = w.clone()
    _overwrite()
    for a, c in zip(want, torch.autograd.grad(loss, (x, p))):
        assert torch.equal(a, c)
