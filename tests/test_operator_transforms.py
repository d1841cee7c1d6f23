"""Forward-mode derivatives of packed attention, layer norm and the top-logits KL are refused
like those of the framework's other operators: a tangent never gets lost on the way. Without
a GPU the kernels' calls are replaced, so the path to them is what is tested."""

import pytest
import torch
import torch.autograd.forward_ad as fw

from param_decomp_amd import losses, ops
from param_decomp_amd.attention import packed_attention
from param_decomp_amd.norms import layer_norm


def _calls(device):
    """(call, its differentiable inputs) of each operator."""
    q, k = torch.randn(6, 4, 16, device=device), torch.randn(6, 2, 16, device=device)
    off = torch.tensor([0, 2, 6], dtype=torch.int32, device=device)
    x, w = torch.randn(3, 8, device=device), torch.ones(8, device=device)
    idx = torch.zeros(3, 2, dtype=torch.int64, device=device)
    return [
        (lambda q, k, v: packed_attention(q, k, v, off), [q, k, k.clone()]),
        (lambda q, k, v: packed_attention(q, k, v, off), [t[..., :12] for t in (q, k, k.clone())]),  # padded widths
        (lambda x, w, b: layer_norm(x, w, b), [x, w, w.clone()]),
        (lambda z: losses.top_logits_position_kl(z, x[:, :2], idx), [x.clone()]),
        (lambda z: losses.top_logits_kl(z, x[:, :2], idx), [x.clone()]),
    ]


def _refuse_tangents(device):
    for call, inputs in _calls(device):
        for i, t in enumerate(inputs):
            for grad in (True, False):
                with fw.dual_level(), torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="jvp"):
                    call(*inputs[:i], fw.make_dual(t, torch.ones_like(t)), *inputs[i + 1:])
        with fw.dual_level():  # no tangent, no refusal
            assert call(*inputs).grad_fn is None
        leaf = inputs[0].detach().clone().requires_grad_()
        assert call(leaf, *inputs[1:]).grad_fn is not None
        with torch.no_grad():
            assert call(leaf, *inputs[1:]).grad_fn is None


def test_tangents_are_refused(monkeypatch):
    monkeypatch.setattr(ops, "packed_attention_fwd", lambda q, k, v, off, scale=None, want_saved=False:
                        (torch.zeros_like(q), (q.new_zeros(1), None) if want_saved else None))
    monkeypatch.setattr(ops, "layer_norm_fwd", lambda x, w=None, b=None, eps=1e-5, want_stats=False:
                        (torch.zeros_like(x), x.new_zeros(1)))
    monkeypatch.setattr(ops, "top_logits_kl", lambda z, top, idx, **kw: (z.new_zeros(z.shape[:-1]), None))
    _refuse_tangents("cpu")


@pytest.mark.gpu
def test_tangents_are_refused_on_the_gpu(device):
    _refuse_tangents(device)
