"""expert_mlp on the CPU: the operators' composition, and what the call and its C entry point refuse."""

import ctypes

import pytest
import torch
import torch.nn.functional as F

import adambridge_amd as ab
from adambridge_amd import _hip


def _operands(gen, dtype=torch.float64):
    return [torch.randn(*s, generator=gen, dtype=dtype) for s in ((7, 6), (7, 4), (4, 5, 6), (4, 6, 5), (4, 5, 6))]


@pytest.mark.parametrize("activation", ["gelu", "silu"])
@pytest.mark.parametrize("gated", [False, True])
def test_the_loop_over_tokens(gated, activation):
    x, logits, up, down, gate = _operands(torch.Generator().manual_seed(0))
    got = ab.expert_mlp(x, logits, up, down, 2, gate if gated else None, activation)
    act = F.gelu if activation == "gelu" else F.silu
    for t in range(7):
        weights, chosen = torch.topk(logits[t], 2)
        want = 0.0
        for w, e in zip(torch.softmax(weights, 0), chosen):
            h = up[e] @ x[t]
            want = want + w * (down[e] @ (act(gate[e] @ x[t]) * h if gated else act(h)))
        assert torch.allclose(got[t], want)


def test_gradients():
    x, logits, up, down, gate = (t.requires_grad_() for t in _operands(torch.Generator().manual_seed(1)))
    assert torch.autograd.gradcheck(lambda *a: ab.expert_mlp(*a[:4], 2, a[4], "silu"), (x, logits, up, down, gate))


def test_refusals():
    x, logits, up, down, gate = _operands(torch.Generator().manual_seed(2), torch.float32)
    for call, words in (
            (lambda: ab.expert_mlp(x, logits, up, down, 2, activation="relu"), "activation must be one of gelu, silu"),
            (lambda: ab.expert_mlp(x[0], logits, up, down, 2), r"x \[tokens, hidden\]"),
            (lambda: ab.expert_mlp(x[:5], logits, up, down, 2), r"x \[tokens, hidden\]"),
            (lambda: ab.expert_mlp(x, logits[:, :3], up, down, 2), r"up \[experts, inter, hidden\]"),
            (lambda: ab.expert_mlp(x, logits, up[:, :, :5], down, 2), r"up \[experts, inter, hidden\]"),
            (lambda: ab.expert_mlp(x, logits, up, down.transpose(1, 2), 2), r"down must be \[experts, hidden, inter\]"),
            (lambda: ab.expert_mlp(x, logits, up, down, 2, gate[:, :4]), "gate, if any, as up"),
            (lambda: ab.expert_mlp(x, logits, up.double(), down, 2), "of one type"),
            (lambda: ab.expert_mlp(x, logits, up, down, 2, gate.bfloat16()), "of one type"),
            (lambda: ab.expert_mlp(x, logits, up, down, 5), "top_k must be an int"),
            (lambda: ab.expert_mlp(x, logits, up, down, True), "top_k must be an int")):
        with pytest.raises(ValueError, match=words):
            call()


def test_entry_point():
    lib, p, f32 = _hip.open_library(), ctypes.c_void_p(256), _hip.DT_F32
    mlp, work = lib.adambridge_expert_mlp, lib.adambridge_expert_mlp_work
    for sizes in ((0, 4, 2, 8, 8), (17, 4, 2, 8, 8), (4, 0, 1, 8, 8), (4, 1025, 2, 8, 8), (4, 4, 0, 8, 8), (4, 4, 5, 8, 8), (4, 100, 65, 8, 8),
                  (4, 4, 2, 0, 8), (4, 4, 2, 8, 0), (4, 4, 2, (1 << 22) + 1, 8), (4, 4, 2, 8, (1 << 22) + 1)):
        assert mlp(p, p, f32, p, None, p, f32, *sizes, 0, 1, p, p) == -1 and work(f32, *sizes) == -1
    sizes = (4, 4, 2, 8, 8)
    assert mlp(p, p, _hip.DT_FP8, p, None, p, f32, *sizes, 0, 1, p, p) == -4
    assert mlp(p, p, f32, p, None, p, _hip.DT_FP8, *sizes, 0, 1, p, p) == -4 and work(_hip.DT_FP8, *sizes) == -4
    assert mlp(p, p, f32, p, None, p, f32, *sizes, 2, 1, p, p) == -4 and mlp(p, p, f32, p, None, p, f32, *sizes, -1, 1, p, p) == -4
    for i in (0, 1, 3, 5, 14, 15):
        args = [p, p, f32, p, None, p, f32, *sizes, 0, 1, p, p]
        args[i] = None
        assert mlp(*args) == -2
    assert mlp(p, p, f32, p, None, p, f32, *sizes, 0, 1, p, ctypes.c_void_p(264)) == -14
    assert work(f32, 16, 64, 8, 100, 8) > 64 * 16 * 100 * 4 and work(f32, 1, 64, 8, 100, 8) < 9 * 16 * 100 * 4


def _copies(monkeypatch, call):
    """The tensors that expert_mlp itself lays out again in ``call``, with its conditions taken as on a GPU."""
    import sys

    from adambridge_amd import experts

    class Native:
        def __getattr__(self, name):
            return lambda *args: None   # every kernel declines: torch operations

    seen, contiguous = [], torch.Tensor.contiguous

    def counted(self, *args, **kwargs):
        if sys._getframe(1).f_code is experts.expert_mlp.__code__:
            seen.append(self)
        return contiguous(self, *args, **kwargs)

    with monkeypatch.context() as m:
        m.setattr(experts, "plain", lambda *ts: all(t is None or t.dtype in (torch.float32, torch.bfloat16) for t in ts))
        m.setattr(experts._hip, "ops", lambda: Native())
        m.setattr(torch.Tensor, "contiguous", counted)
        call()
    return seen


def test_operands_are_laid_out_again_only_for_a_call_that_the_kernels_take(monkeypatch):
    """A trained call, one under autocast or observed, one of many tokens or of sizes that they do not take: expert_mm lays out what
    it needs, and nothing is copied twice."""
    x, logits, up, down, gate = _operands(torch.Generator().manual_seed(3), torch.float32)
    strided = up.transpose(1, 2).contiguous().transpose(1, 2)
    call = lambda *more, x=x, logits=logits, up=strided, down=down, top_k=2: lambda: ab.expert_mlp(x, logits, up, down, top_k, *more)
    assert len(_copies(monkeypatch, call())) == 4 and len(_copies(monkeypatch, call(gate))) == 5
    assert not _copies(monkeypatch, call(up=up))
    for leaf in (x, logits, strided, down, gate):
        leaf.requires_grad_()
        assert not _copies(monkeypatch, call(gate))
        with torch.no_grad():
            assert len(_copies(monkeypatch, call(gate))) == 5
        leaf.requires_grad_(False)
    with torch.autocast("cpu", dtype=torch.bfloat16):
        assert not _copies(monkeypatch, call())
    assert not _copies(monkeypatch, lambda: torch.func.vmap(lambda t: ab.expert_mlp(t, logits, strided, down, 2))(torch.stack((x, x))))
    assert not _copies(monkeypatch, call(x=torch.cat((x, x, x)), logits=torch.cat((logits, logits, logits))))
    assert not _copies(monkeypatch, call(x=x[:0], logits=logits[:0]))
    half = [t.half() for t in (x, strided, down)]
    assert not _copies(monkeypatch, call(x=half[0], up=half[1], down=half[2]))
    wide = [torch.randn(*s) for s in ((2, 6), (2, 1030), (1030, 1, 6), (1030, 6, 1))]
    assert not _copies(monkeypatch, call(x=wide[0].t().contiguous().t(), logits=wide[1], up=wide[2], down=wide[3]))
    assert not _copies(monkeypatch, call(x=wide[0].t().contiguous().t(), logits=wide[1][:, :70], up=wide[2][:70], down=wide[3][:70], top_k=65))
    with pytest.raises(ValueError, match="top_k must be an int"):
        _copies(monkeypatch, call(top_k=True))
