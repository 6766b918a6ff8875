"""Calls of kernels without a backward pass refuse every tensor whose gradient they would lose, in either mode of differentiation."""
import pytest
import torch
from torch.autograd import forward_ad

from gaac_amd import FP4KVCache, qk_norm_rope

BF = torch.bfloat16


def calls(device):
    """name -> call(t), t being applied to one of the call's tensors."""
    x, pos, w = torch.zeros(5, 2, 128, dtype=BF, device=device), torch.zeros(5, dtype=torch.int64, device=device), torch.ones(128, dtype=BF, device=device)
    cos, slots = torch.zeros(10, 64, device=device), torch.arange(5, dtype=torch.int32, device=device)
    c = FP4KVCache(5, 2, 64, device=device)
    return {
        "prefill k": lambda t: c.prefill(0, t(x), x), "prefill v": lambda t: c.prefill(0, x, t(x)), "append k": lambda t: c.append(slots, t(x), x), "append v": lambda t: c.append(slots, x, t(x)),
        "attention q": lambda t: c.attention(t(x), slots, 1.0), "attention q, splits": lambda t: c.attention(t(x), slots, 1.0, nsplit=2),
        "rotation q": lambda t: qk_norm_rope(t(x), x, pos, cos, cos), "rotation k": lambda t: qk_norm_rope(x, t(x), pos, cos, cos),
        "rotation cos": lambda t: qk_norm_rope(x, x, pos, t(cos), cos), "rotation sin": lambda t: qk_norm_rope(x, x, pos, cos, t(cos)),
        "rotation q_weight": lambda t: qk_norm_rope(x, x, pos, cos, cos, t(w), w), "rotation k_weight": lambda t: qk_norm_rope(x, x, pos, cos, cos, w, t(w)),
    }


def check(device, name, runs):
    """runs(call): makes a call that has nothing to refuse."""
    call = calls(device)[name]
    need = lambda t: t.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="no backward pass"): call(need)
    with torch.no_grad(): runs(lambda: call(need))
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t.clone(), torch.ones_like(t))
        with pytest.raises(RuntimeError, match="no backward pass"): call(dual)
        with torch.no_grad(), pytest.raises(RuntimeError, match="no backward pass"): call(dual)      # (which leaves the other mode on)
        runs(lambda: call(lambda t: t))
    runs(lambda: call(lambda t: t))


def no_device(f):
    with pytest.raises(RuntimeError, match="no CPU path"): f()


@pytest.mark.parametrize("name", calls("cpu"))
def test_on_the_host(name): check("cpu", name, no_device)


@pytest.mark.gpu
@pytest.mark.parametrize("name", calls("cpu"))
def test_on_the_device(name):
    from gpu_util import require_gpu
    require_gpu()
    check("cuda", name, lambda f: f())
