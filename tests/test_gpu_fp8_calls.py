"""The calls of rows and weights in 8 bits and of log probabilities that the binding makes as a whole against the same calls through Python; on streams of their own, and captured in graphs."""
import pytest
import torch

from gaac_amd import FP8Rows, FP8Weight, _lib, fp8_gated, fp8_linear, quantize_fp8, rms_norm_fp8, token_logprobs
from gpu_util import require_gpu

pytestmark = pytest.mark.gpu
WHOLE = ("fp8_rows", "fp8_multiply", "fp8_values", "logprobs")


@pytest.fixture
def both(monkeypatch):
    """both(f): f's results with the binding and with Python's calls, and of each whole call that f came to whether the binding made it."""
    require_gpu()
    binding = _lib.calls()
    assert hasattr(binding, "bind")
    def run(f):
        out, made = [], []
        class Watched:
            def __getattr__(self, name):
                def call(*a):
                    r = getattr(binding, name)(*a)
                    if name in WHOLE: made.append(r is not None)
                    return r
                return call
        for calls in (Watched(), _lib._CtypesCalls()):
            monkeypatch.setattr(_lib, "_calls", calls)
            try: out.append(f())
            except (RuntimeError, TypeError) as e: out.append((type(e), str(e)))
        monkeypatch.setattr(_lib, "_calls", binding)
        return out[0], out[1], made
    return run


def rnd(*shape, seed=0, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def same(a, b):
    assert type(a) is type(b)
    if isinstance(a, torch.Tensor): assert a.dtype == b.dtype and a.stride() == b.stride() and torch.equal(a, b)
    elif isinstance(a, FP8Rows): assert a.shape == b.shape; same(a.dequantize(), b.dequantize())
    elif isinstance(a, (tuple, list)):
        assert len(a) == len(b)
        for x, y in zip(a, b): same(x, y)
    else: assert a == b


FORMS = {      # rows -> (a view of it, whether the binding takes it)
    "plain": (lambda x: x, True), "one row": (lambda x: x[:1], True), "wide stride": (lambda x: x[:, 16:144], True), "odd columns": (lambda x: x[:, 3:100], True), "every other": (lambda x: x[::2], True),
    "one row for all": (lambda x: x[:1].expand(20, 160), True), "columns apart": (lambda x: x[:, ::2], False), "none": (lambda x: x[:0], False), "no rows": (lambda x: x[0], False), "wrong type": (lambda x: x.double(), False),
}


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_calls_are_the_same_both_ways(both, form, dtype):
    view, whole = FORMS[form]
    x = view(rnd(20, 160, seed=1, dtype=dtype))
    K = x.shape[-1]
    w, up, g, r = rnd(40, K, seed=2), rnd(40, K, seed=3), rnd(K, seed=4, dtype=dtype), view(rnd(20, 160, seed=5, dtype=dtype))
    W, G = FP8Weight(w), FP8Weight(w, up)
    tokens = torch.arange(len(x), device="cuda")
    for f in (lambda: quantize_fp8(x), lambda: rms_norm_fp8(x, g), lambda: rms_norm_fp8(x, g, 1e-5, residual=r), lambda: fp8_linear(x, W), lambda: fp8_linear(x, W, out_dtype=torch.float32), lambda: fp8_gated(x, G),
              lambda: fp8_gated(x, G, quantize=True), lambda: token_logprobs(x, tokens), lambda: token_logprobs(x, tokens, top=7)):
        a, b, made = both(f)
        same(a, b)
        assert not made or all(made) == whole      # (no call: the arguments were refused before)


def test_what_is_refused_is_refused_both_ways(both):
    x, w, t = rnd(5, 256), FP8Weight(rnd(64, 256)), torch.arange(5, device="cuda")
    need = rnd(5, 256).requires_grad_()
    for f in (lambda: fp8_linear(x, FP8Weight(rnd(64, 128))), lambda: fp8_gated(x, w), lambda: fp8_linear(x, w, out_dtype=torch.float64), lambda: quantize_fp8(need), lambda: fp8_linear(need, w),
              lambda: rms_norm_fp8(x, need[0]), lambda: rms_norm_fp8(x, x[0], residual=need), lambda: rms_norm_fp8(x, x[0], residual=x[:4]), lambda: token_logprobs(need, t), lambda: token_logprobs(x, t.int()),
              lambda: token_logprobs(x, t, top=65), lambda: fp8_linear(x.cpu(), w), lambda: token_logprobs(x, t.cpu()), lambda: rms_norm_fp8(x, x[0].cpu())):
        a, b, _ = both(f)
        assert a == b and a[0] is RuntimeError, a


def test_integers_for_eps_and_detached_gradients(both):
    x, need = rnd(5, 256), rnd(5, 256).requires_grad_()
    same(*both(lambda: rms_norm_fp8(x, x[0], 0))[:2])
    with torch.no_grad(): same(*both(lambda: quantize_fp8(need))[:2])


def test_streams_and_graphs():
    """Calls on a stream of their own, captured and replayed with other inputs, with eager calls between the replays."""
    require_gpu()
    M, K, F, V = 40, 512, 384, 20000
    x, r, g = rnd(M, K, seed=1), rnd(M, K, seed=2), rnd(K, seed=3)
    W, G, D, head = FP8Weight(rnd(K, K, seed=4)), FP8Weight(rnd(F, K, seed=5), rnd(F, K, seed=6)), FP8Weight(rnd(K, F, seed=7)), FP8Weight(rnd(V, K, seed=8))
    tokens = torch.arange(M, device="cuda") * 7
    def layer():
        rows, h = rms_norm_fp8(x, g, 1e-5, residual=r)
        o = fp8_linear(rows, W)
        y = fp8_linear(fp8_gated(o, G, quantize=True), D)
        return [h, o, y, *token_logprobs(fp8_linear(y, head, out_dtype=torch.float32), tokens, top=5)]
    want = layer()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = layer()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side): held = layer()
    torch.cuda.current_stream().wait_stream(side)
    same(want, other)
    for i in range(4):
        x.copy_(rnd(M, K, seed=20 + i))
        want = layer()
        graph.replay()
        torch.cuda.synchronize()
        same(want, held)
        layer()
