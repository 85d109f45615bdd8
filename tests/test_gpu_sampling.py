"""The next token of every row, against its definition in float64. Weights are multiples of 2^-44
of the largest at the least, so a row's sums err by under vocabulary * 2^-45 of it: up to 2^-27. Tokens
are whole numbers and have to be equal; draws of u so near a border that float64 could
round to the other side are told from the oracle alone, and there are none among these."""
import numpy as np
import pytest
import torch

from oracle import sample_oracle as O

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def sampling():
    from perm_amd import sampling
    return sampling


def _check(sampling, logits, u, **settings):
    """One call with per-row settings where they are lists; every row against the oracle."""
    rows = logits.shape[0]
    args, each = {}, [dict() for _ in range(rows)]
    for name, v in settings.items():
        if isinstance(v, (list, tuple, np.ndarray)):
            t = torch.tensor(v, dtype=torch.int32 if name == "top_k" else torch.float32)
            args[name] = t.cuda()
            v = t.tolist()
        else:
            args[name] = v
            v = [v] * rows
        for r in range(rows):
            each[r][name] = v[r]
    got = sampling.sample(logits, u, **args).cpu().tolist()
    x, u = logits.double().cpu().numpy(), u.double().cpu().numpy()
    for r in range(rows):
        want, near = O.sample(x[r], u[r], **each[r])
        assert got[r] == want, (r, got[r], want, near, each[r])


def _logits(seed, rows, vocab, dtype, scale=2.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((rows, vocab), generator=g, device="cuda") * scale
    return x.to(dtype), torch.rand((rows,), generator=g, device="cuda")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 63, 100, 512, 1000, 1025, 8191, 32001, 151936])
def test_sizes(sampling, vocab, dtype):
    print(f"sample {vocab} {dtype}", flush=True)
    x, u = _logits(vocab, 12, vocab, dtype)
    _check(sampling, x, u, temperature=[0.0, 0.3, 1.0, 1.5, 0.7, 1.0, 1.0, 2.0, 1.0, 1.0, 30.0, 0.01],
           top_k=[0, 0, 0, 0, 1, 50, 0, 1000, 40, 5000, 0, 3],
           top_p=[1.0, 0.9, 1.0, 0.95, 1.0, 0.9, 0.5, 0.99, 1.0, 0.8, 0.7, 1.0],
           min_p=[0.0, 0.0, 0.0, 0.05, 0.0, 0.0, 0.0, 0.001, 0.2, 0.0, 0.0, 0.0])
    _check(sampling, x, u)
    _check(sampling, x, u, temperature=0.7, top_k=50, top_p=0.9, min_p=0.01)


@pytest.mark.parametrize("dtype", DTYPES)
def test_every_border_of_a_cut(sampling, dtype):
    """top_k at every size around the list's and the histogram's; all of them at once."""
    x, u = _logits(5, 24, 40000, dtype, 1.0)
    k = [1, 2, 3, 63, 64, 65, 127, 500, 1000, 1023, 1024, 1025, 1500, 2047, 2048, 2049, 4096, 9999, 20000,
         39998, 39999, 40000, 40001, 2 ** 31 - 1]
    _check(sampling, x, u, top_k=k)
    _check(sampling, x, u, top_k=k, top_p=0.6)
    _check(sampling, x, u, top_k=k, top_p=0.97, min_p=0.05, temperature=1.3)
    p = np.linspace(0, 1, 24)
    _check(sampling, x, u, top_p=p)
    _check(sampling, x, u, min_p=p)


def test_equal_logits_go_by_number(sampling):
    """Few values, many of each: cuts inside runs of equal logits, and u on the borders themselves."""
    g = torch.Generator(device="cuda").manual_seed(1)
    for values, vocab in ((1, 4096), (2, 5000), (3, 30000), (40, 70000)):
        x = torch.randint(0, values, (16, vocab), generator=g, device="cuda").float()
        u = torch.rand((16,), generator=g, device="cuda")
        for settings in (dict(top_k=7), dict(top_k=1500), dict(top_k=3000, top_p=0.5), dict(top_p=0.3),
                         dict(top_p=0.9, temperature=0.25), dict(min_p=0.5), dict(min_p=1.0), dict(),
                         dict(top_k=[1 + 300 * i for i in range(16)], top_p=0.75)):
            _check(sampling, x, u, **settings)
    # four equal tokens: quarters, exactly
    x = torch.full((8, 9), -30000.0, device="cuda")
    x[:, [1, 4, 5, 8]] = 2.0
    u = torch.arange(8, device="cuda") / 8
    assert sampling.sample(x, u).tolist() == [1, 1, 4, 4, 5, 5, 8, 8]
    assert sampling.sample(x, u, top_p=0.75).tolist() == [1, 1, 1, 4, 4, 4, 5, 5]
    assert sampling.sample(x, u, top_p=0.5).tolist() == [1, 1, 1, 1, 4, 4, 4, 4]
    assert sampling.sample(x, u, top_k=2).tolist() == [1, 1, 1, 1, 4, 4, 4, 4]
    assert sampling.sample(x, u, min_p=1.0).tolist() == [1, 1, 4, 4, 5, 5, 8, 8]


@pytest.mark.parametrize("dtype", DTYPES)
def test_extremes(sampling, dtype):
    """Masked tokens in both customs, NaN, infinities, rows of nothing, zeros of both signs."""
    inf, low, high = float("inf"), torch.finfo(dtype).min, torch.finfo(dtype).max
    x, u = _logits(3, 20, 3000, torch.float32)
    x[0] = -inf
    x[1] = float("nan")
    x[2, 1:] = -inf
    x[3, :2999] = float("nan")
    x[4] = low
    x[5, 100:] = low
    x[6, 200], x[6, 300] = inf, inf
    x[7, 0], x[7, 1] = inf, low
    x[8] = inf
    x[9, ::2] = -inf
    x[10, 5] = high
    x[11] = 0.0
    x[11, ::2] = -0.0
    x[12] = low
    x[12, 77] = high
    x[13, 1] = float("nan")
    x[14] = torch.linspace(-1e-30, 1e-30, 3000)
    x[15] = -inf
    x[15, 1234] = low
    x[16] *= 1e4 if dtype != torch.float16 else 1e3
    x = x.to(dtype)
    for settings in (dict(), dict(top_k=10), dict(top_p=0.9), dict(min_p=0.1), dict(temperature=0.0),
                     dict(top_k=2000, top_p=0.7, min_p=0.01), dict(temperature=1e-30), dict(temperature=1e30),
                     dict(temperature=float("inf"), top_p=0.5), dict(top_k=1), dict(top_p=0.0), dict(top_k=2999)):
        _check(sampling, x, u, **settings)


def test_temperatures_whose_reciprocal_is_no_number(sampling):
    """Numbers for all rows come in double precision: the largest logits alone weigh, all the same."""
    x, u = _logits(11, 6, 5000, torch.float32)
    x[3, [7, 70, 700]] = 100.0
    for t in (5e-324, 1e-320, 1e-308, 1e-291):
        for more in (dict(), dict(top_p=0.9), dict(top_k=5), dict(top_k=2000), dict(min_p=0.5)):
            got = sampling.sample(x, u, temperature=t, **more)
            assert torch.equal(x.gather(1, got.long()[:, None])[:, 0], x.amax(1)), (t, more)
            assert torch.equal(got, sampling.sample(x, u, temperature=1e-30, **more)), (t, more)


def test_numbers_at_the_ends_of_their_range(sampling):
    x, _ = _logits(9, 6, 5000, torch.float32)
    u = torch.tensor([0.0, 1.0 - 2.0 ** -24, 0.5, 0.25, 1.0, float("nan")], device="cuda")
    got = sampling.sample(x, u)
    assert torch.equal(got[:4], sampling.sample(x, u.double())[:4])
    _check(sampling, x[:4], u[:4])
    assert got[5] == 0 and got[4] == 4999  # no number: as 0; 1: the last token
    bad = torch.tensor([-1.0, float("nan"), 2.0, -3.0, 0.5, 1.0], device="cuda")
    as_t = sampling.sample(x, u, temperature=bad)
    assert torch.equal(as_t[[0, 1, 3]], x.argmax(1).to(torch.int32)[[0, 1, 3]])
    clipped = bad.nan_to_num(0.0).clamp(0, 1)
    assert torch.equal(sampling.sample(x, u, min_p=bad), sampling.sample(x, u, min_p=clipped))
    p = bad.nan_to_num(1.0).clamp(0, 1)
    assert torch.equal(sampling.sample(x, u, top_p=bad), sampling.sample(x, u, top_p=p))
    k = torch.tensor([-5, 0, 5000, 6000, -2 ** 31, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    assert torch.equal(sampling.sample(x, u, top_k=k), got)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_alignment(sampling, dtype):
    x, u = _logits(4, 9, 2000, dtype)
    want = sampling.sample(x, u, top_p=0.9)
    wide = torch.full((9, 2003), float("inf"), dtype=dtype, device="cuda")
    for at in range(4):
        wide.fill_(float("inf"))
        wide[:, at:at + 2000] = x
        assert torch.equal(sampling.sample(wide[:, at:at + 2000], u, top_p=0.9), want)
    assert torch.equal(sampling.sample(x.t().contiguous().t(), u, top_p=0.9), want)
    assert torch.equal(sampling.sample(x.repeat_interleave(2, 0)[::2], u, top_p=0.9), want)
    one = x[:1].expand(9, 2000)
    assert torch.equal(sampling.sample(one, u), sampling.sample(one.contiguous(), u))
    s = torch.rand((18,), device="cuda")
    s[::2] = u
    assert torch.equal(sampling.sample(x, s[::2], top_p=0.9), want)


def test_a_row_is_the_same_in_any_batch(sampling):
    x, u = _logits(6, 300, 20000, torch.bfloat16)
    for settings in (dict(top_p=0.9), dict(top_k=40), dict(), dict(top_k=3000, min_p=0.001)):
        want = sampling.sample(x, u, **settings)
        for a, b in ((0, 1), (7, 9), (100, 164), (13, 300)):
            assert torch.equal(sampling.sample(x[a:b], u[a:b], **settings), want[a:b])


def test_draws_follow_the_weights(sampling):
    """Every border hit from both sides: u stepping through a small vocabulary."""
    x, _ = _logits(8, 1, 50, torch.float32, 1.0)
    u = (torch.arange(4096, device="cuda") + 0.5) / 4096
    _check(sampling, x.expand(4096, 50), u, top_p=0.95)


def test_graph_replays(sampling):
    x, u = _logits(10, 40, 33000, torch.bfloat16)
    t = torch.full((40,), 1.0, device="cuda")

    def step():
        return sampling.sample(x, u, temperature=t, top_p=0.9), sampling.sample(x, u, top_k=50), sampling.sample(x, u)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    g = torch.Generator(device="cuda").manual_seed(3)
    for i in range(4):
        graph.replay()
        torch.cuda.synchronize()
        got = [y.clone() for y in outs]
        for a, b in zip(got, step()):
            assert torch.equal(a, b), i
        x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
        u.copy_(torch.rand(u.shape, generator=g, device="cuda"))
        t.mul_(0.8)


def test_two_streams_at_once(sampling):
    x, u = _logits(12, 200, 50000, torch.bfloat16)
    kinds = [dict(top_p=0.9), dict(top_k=50, top_p=0.95), dict(min_p=0.02), dict(top_k=1500)]
    want = [sampling.sample(x, u, **k) for k in kinds]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                got.append([sampling.sample(x, u, **k) for k in kinds])
    torch.cuda.synchronize()
    for tokens in got:
        assert all(torch.equal(a, b) for a, b in zip(tokens, want))


def test_refusals(sampling, monkeypatch):
    x, u = _logits(1, 4, 100, torch.float32)
    with pytest.raises(TypeError):
        sampling.sample(x.double(), u)
    with pytest.raises(TypeError):
        sampling.sample(x, u.half())
    with pytest.raises(TypeError):
        sampling.sample([1.0], u)
    for bad in (dict(temperature=-1.0), dict(temperature=float("nan")), dict(top_k=-1), dict(top_p=1.5),
                dict(top_p=float("nan")), dict(min_p=-0.1), dict(temperature=torch.ones(4)),
                dict(temperature=torch.ones(3, device="cuda")), dict(top_k=torch.ones(4, device="cuda"))):
        with pytest.raises(ValueError):
            sampling.sample(x, u, **bad)
    with pytest.raises(TypeError):
        sampling.sample(x, u, top_k=1.5)
    for args in ((x.cpu(), u), (x, u.cpu()), (x[0], u), (x, u[:3]), (x[:, :0], u)):
        with pytest.raises(ValueError):
            sampling.sample(*args)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    with pytest.raises(ValueError, match="current device"):
        sampling.sample(x, u)
    monkeypatch.undo()
    assert sampling.sample(x[:0], u[:0]).shape == (0,)
