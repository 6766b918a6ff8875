"""The calls of the 4-bit cache, of qk_norm_rope and of sample that the binding makes as a whole against the same calls through Python, over the forms that either takes, on
streams of their own and with what is refused; and which of them the binding makes."""
import pytest
import torch

from gaac_amd import FP4KVCache, _lib, qk_norm_rope, sample
from gpu_util import require_gpu

pytestmark = pytest.mark.gpu
WHOLE = ("fp4_prefill", "fp4_append", "fp4_attend", "fp4_read", "norm_rope", "draw")


@pytest.fixture
def both(monkeypatch):
    """both(f): f's results with the binding and with Python's calls, and for each whole call that f came to, whether the binding made it."""
    require_gpu()
    binding = _lib.calls()
    assert hasattr(binding, "bind")
    def run(f):
        out, made = [], {}
        class Watched:
            def __getattr__(self, name):
                def call(*a):
                    r = getattr(binding, name)(*a)
                    if name in WHOLE: made.setdefault(name, []).append(r is not None)
                    return r
                return call
        for calls in (Watched(), _lib._CtypesCalls()):
            monkeypatch.setattr(_lib, "_calls", calls)
            try: out.append(f())
            except (RuntimeError, TypeError) as e: out.append((type(e), str(e)))
        monkeypatch.setattr(_lib, "_calls", binding)
        return out[0], out[1], made
    return run


def same(a, b):
    assert type(a) is type(b)
    if isinstance(a, torch.Tensor): assert a.dtype == b.dtype and torch.equal(a, b)
    elif isinstance(a, (tuple, list)):
        assert len(a) == len(b)
        for x, y in zip(a, b): same(x, y)
    else: assert a == b


def rnd(*shape, seed=0, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


FORMS = {
    "plain": (lambda n, h, seed: rnd(n, h, 128, seed=seed), True),
    "of a projection": (lambda n, h, seed: rnd(n, h + 3, 128, seed=seed)[:, 2:2 + h], True),
    "head-major": (lambda n, h, seed: rnd(h, n, 128, seed=seed).transpose(0, 1), True),
    "misaligned": (lambda n, h, seed: rnd(n * h * 128 + 1, seed=seed)[1:].view(n, h, 128), False),
    "every other channel": (lambda n, h, seed: rnd(n, h, 256, seed=seed)[..., ::2], False),
    "another type": (lambda n, h, seed: rnd(n, h, 128, seed=seed, dtype=torch.float64), False),
    "other heads": (lambda n, h, seed: rnd(n, h + 1, 128, seed=seed), None),
}


@pytest.mark.parametrize("form", FORMS)
def test_the_cache(both, form):
    make, whole = FORMS[form]
    def steps():
        c = FP4KVCache(3, 2, 1700)
        k, v = make(1650, 2, 1), make(1650, 2, 2)
        c.prefill(1, k, v)
        slots = torch.tensor([1, -1, 2], dtype=torch.int32, device="cuda")
        c.append(slots, make(3, 2, 3), make(3, 2, 4))
        q = rnd(3, 8, 128, seed=5)
        return c.data, c.lens, c.attention(q, slots, 0.1), c.attention(q, slots, 1, max_len=1700, nsplit=5), c.attention(q[:, ::2], slots, 0.1), c.decompress(1), c.decompress(0), c.stats()
    a, b, made = both(steps)
    same(a, b)
    if whole is None or form == "another type": assert isinstance(a[0], type) and issubclass(a[0], RuntimeError) and "bf16" in a[1]
    else: assert made == dict(fp4_prefill=[whole], fp4_append=[whole], fp4_attend=[True, False, False], fp4_read=[True, True])


@pytest.mark.parametrize("form", FORMS)
def test_norm_and_rotation(both, form):
    make, whole = FORMS[form]
    pos, cos = torch.arange(20, device="cuda") * 3, rnd(70, 64, dtype=torch.float32)
    w = rnd(128, seed=9)
    for args in ((), (w, w), (w, torch.stack([w] * 2))):
        a, b, made = both(lambda: qk_norm_rope(make(20, 5, 1), make(20, 2, 2), pos, cos, cos, *args, eps=1e-5))
        same(a, b)
        if form == "another type" or form == "other heads" and len(args) and args[1].dim() == 2: assert issubclass(a[0], RuntimeError)
        else: assert made == dict(norm_rope=[whole is not False])
    a, b, made = both(lambda: qk_norm_rope(rnd(20, 5, 128), rnd(20, 2, 128), pos, cos.t().contiguous().t(), cos, eps=0))
    same(a, b)
    assert made == dict(norm_rope=[False])


@pytest.mark.parametrize("V", [100, 6000])
def test_sampling(both, V):
    x, u = rnd(5, 2 * V, seed=1), torch.rand(5, generator=torch.Generator().manual_seed(2)).cuda()
    rows = dict(temperature=torch.full((5,), 0.7, device="cuda"), top_k=torch.arange(5, dtype=torch.int32, device="cuda"), top_p=torch.full((5,), 0.9, device="cuda"), min_p=torch.zeros(5, device="cuda"))
    for logits, settings, whole in ((x, {}, True), (x, dict(temperature=1, top_k=3, top_p=1), True), (x, rows, True), (x[:, V // 2:V + 3], rows, True), (x[::2], dict(top_p=0.9), True), (x[:, ::2], rows, False), (x, dict(top_k=3.0), False),
                                    (x, dict(top_k=10 ** 12), True), (x[:0], {}, False)):
        a, b, made = both(lambda: sample(logits, u[:logits.shape[0]], **settings))
        same(a, b)
        assert isinstance(a, torch.Tensor) and made == dict(draw=[whole])
    for bad in (dict(top_k=rows["top_p"]), dict(temperature=rows["temperature"][:3]), dict(min_p=rows["min_p"].cpu())):
        a, b, _ = both(lambda: sample(x, u, **bad))
        same(a, b)
        assert issubclass(a[0], RuntimeError)


def test_calls_on_a_stream_of_their_own():
    """Everything a step does on another stream than the default one, behind work that the stream still has to do."""
    require_gpu()
    def step(busy):
        c = FP4KVCache(2, 2, 1700)
        x = torch.zeros(1650, 12, 128, dtype=torch.bfloat16, device="cuda")
        if busy: torch.cuda._sleep(20_000_000)
        x.copy_(rnd(1650, 12, 128))      # what the calls read comes late
        pos, cos = torch.arange(1650, device="cuda"), torch.ones(1650, 64, device="cuda")
        q, k = qk_norm_rope(x[:, :8], x[:, 8:10], pos, cos, cos)
        c.prefill(0, k, x[:, 10:])
        slots = torch.zeros(1, dtype=torch.int32, device="cuda")
        c.append(slots, k[5:6], x[7:8, 10:])
        o = c.attention(q[:1], slots, 0.1)
        token = sample(o.view(1, -1), torch.full((1,), 0.5, device="cuda"), top_p=0.9)
        return q, k, c.data, o, token, c.decompress(0)
    want = step(False)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(True)
        side.synchronize()
    same(list(got), list(want))
