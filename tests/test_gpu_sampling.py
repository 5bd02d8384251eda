"""Sampling on the GPU against the float64 oracle (oracle/sampling.py): the same token,
wherever no decision of the row lies within 2^-36 of its border (weights are integers of
2^-38 at worst and sums of them exact; fp64's own roundings are under 2^-44)."""
import numpy as np
import pytest

from oracle.sampling import sample_row

pytestmark = pytest.mark.gpu

NEAR = 2.0 ** -36


def say(msg):
    print(f"[gpu-case] {msg}", flush=True)


def _run(logits, u, dt="f32", **params):
    """(tokens, the logits that the call read)"""
    import torch

    from deltafin_amd import sampling
    l = torch.from_numpy(np.asarray(logits, np.float32)).cuda()
    if dt == "bf16":
        l = l.bfloat16()
    kw = {k: torch.from_numpy(np.asarray(v, np.int32 if k == "top_k" else np.float32)).cuda()
          for k, v in params.items()}
    out = sampling.sample(l, torch.from_numpy(np.asarray(u, np.float32)).cuda(), **kw)
    torch.cuda.synchronize()
    return out.cpu().numpy(), l.float().cpu().numpy()


def _compare(logits, u, dt="f32", **params):
    found, read = _run(logits, u, dt, **params)
    sure = 0
    for i in range(len(u)):
        one = {k: (int(v[i]) if k == "top_k" else float(np.float32(v[i])))
               for k, v in params.items()}
        want, margin = sample_row(read[i], float(np.float32(u[i])), **one)
        if margin > NEAR:
            sure += 1
            assert found[i] == want, (i, found[i], want, margin, one)
    assert sure >= 0.9 * len(u)
    return found


def _params(rng, rows, vocab):
    pick = lambda p: rng.random(rows) < p
    return dict(temperature=rng.uniform(0.3, 2.0, rows) * ~pick(0.1),
                top_k=np.exp(rng.uniform(0, np.log(vocab + 1), rows)).astype(np.int32) * ~pick(0.3),
                top_p=np.where(pick(0.3), 1.0, rng.uniform(0.05, 1.0, rows)),
                min_p=rng.uniform(0, 0.3, rows) * pick(0.5))


@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (40, 5), (17, 1000), (5, 4096), (24, 4099),
                                        (9, 20001), (3, 131072), (2, 150001)])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_sampling(gpu, rows, vocab, dt):
    rng = np.random.default_rng(rows * 7 + vocab)
    say(f"sample {rows}x{vocab} {dt}")
    for spread in (0.02, 2.5, 30.0):
        l = spread * rng.standard_normal((rows, vocab))
        _compare(l, rng.random(rows), dt, **_params(rng, rows, vocab))
        _compare(l, rng.random(rows), dt)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("name", ["temperature", "top_k", "top_p", "min_p"])
def test_each_limit_alone(gpu, dt, name):
    rng = np.random.default_rng(3)
    rows, vocab = 33, 5003
    l = 3 * rng.standard_normal((rows, vocab))
    say(f"{name} alone {dt}")
    _compare(l, rng.random(rows), dt, **{name: _params(rng, rows, vocab)[name]})


def test_equal_logits(gpu):
    """Weights of one, so that every sum is a whole number of them: u (i + 1/2) / kept draws
    token i, whatever the limits, with ties cut by index."""
    vocab = 5000
    say("equal logits")
    i = np.array([0, 1, 63, 64, 999, 1000, 2499])
    l = np.full((len(i), vocab), -3.25)
    for kept, kw in ((vocab, {}), (2500, dict(top_k=2500)), (2500, dict(top_p=0.5)),
                     (2500, dict(top_p=0.5, min_p=1.0)), (2500, dict(min_p=0.7, top_k=2500))):
        params = {k: np.full(len(i), v) for k, v in kw.items()}
        found, _ = _run(l, (i + 0.5) / kept, **params)
        assert np.array_equal(found, i), kw
    # the two zeros are equal
    l = np.where(np.arange(vocab) % 2 == 0, -0.0, 0.0)[None].repeat(len(i), 0)
    found, _ = _run(l, (i + 0.5) / 2500, top_k=np.full(len(i), 2500))
    assert np.array_equal(found, i)


@pytest.mark.parametrize("tied", [1, 2, 63, 64, 65, 255, 256, 257, 1000, 4095, 4097])
def test_groups_of_equal_logits(gpu, tied):
    """`tied` equal logits among masked ones, at places that no order of the threads gives, a
    neighbouring value in the same range half as often and a far smaller one.  All weights
    but the far one's, e^-61, are equal to 2^-22, so u in the middle of a token's share
    draws that token: over at most 6145 tokens their differences and u's own rounding move a
    border by under 6145 (2^-22 + 2^-25) = 0.002 of a share."""
    say(f"{tied} equal logits")
    rng = np.random.default_rng(tied)
    vocab = 9001
    at = rng.permutation(vocab)
    high, low = np.sort(at[:tied]), np.sort(at[tied:tied + tied // 2])
    order = np.concatenate([high, low])
    draws = np.unique(np.concatenate([[0, tied - 1, len(order) - 1],
                                      rng.integers(0, len(order), 9)]))
    l = np.full((len(draws), vocab), -np.inf)
    l[:, high] = 1.0
    l[:, low] = 1.0 - 2.0 ** -22
    l[:, at[-1]] = -60.0
    u = (draws + 0.5) / len(order)
    found, _ = _run(l, u)
    assert np.array_equal(found, order[draws])
    # the same cut behind the equal ones, by count
    inside = draws[draws < tied]
    found, _ = _run(l[:len(inside)], (inside + 0.5) / tied, top_k=np.full(len(inside), tied))
    assert np.array_equal(found, high[inside])


def test_masked_and_special(gpu):
    say("masked and special")
    rng = np.random.default_rng(4)
    vocab = 4500
    l = rng.standard_normal((9, vocab)).astype(np.float32)
    l[0] = -np.inf                       # nothing left
    l[1] = np.nan
    l[2] = -np.inf
    l[2, 4321] = -5                      # one left
    l[3, ::2] = np.nan
    l[4, 1000:] = -np.inf
    l[5] = np.finfo(np.float32).min      # the type's lowest everywhere: equal weights
    l[6, [7, 4400]] = np.inf
    l[7] = np.finfo(np.float32).min
    l[7, 17] = np.finfo(np.float32).max
    l[8] = -np.inf
    l[8, [3, 9]] = np.finfo(np.float32).min
    for u in (0.0, 0.3, 0.77, 1 - 2.0 ** -24):
        uu = np.full(9, u)
        for kw in ({}, dict(top_k=np.full(9, 2000)), dict(top_p=np.full(9, 0.8)),
                   dict(min_p=np.full(9, 0.2)), dict(temperature=np.zeros(9)),
                   dict(temperature=np.full(9, 1e-30)), dict(temperature=np.full(9, np.inf)),
                   dict(temperature=np.full(9, 1e-30), top_p=np.full(9, 0.9))):
            found, read = _run(l, uu, **kw)
            for r in range(9):
                want, margin = sample_row(read[r], u, **{k: v[r] for k, v in kw.items()})
                if margin > NEAR:
                    assert found[r] == want, (r, u, kw, found[r], want)
            assert found[0] == -1 and found[1] == -1 and found[2] == 4321
            assert found[6] in (7, 4400) and found[7] == 17 or "temperature" in kw


def test_parameters_out_of_range(gpu):
    """Values at and past each end mean what the interface says."""
    say("out of range")
    rng = np.random.default_rng(5)
    rows, vocab = 6, 4200
    l = rng.standard_normal((rows, vocab)).astype(np.float32)
    u = np.array([0.1, 0.4, 0.6, 0.9, 0.99, 0.5], np.float32)
    base, _ = _run(l, u)
    same = lambda **kw: np.array_equal(_run(l, u, **{k: np.full(rows, v) for k, v in kw.items()})[0],
                                       base)
    assert same(top_k=0) and same(top_k=-5) and same(top_k=vocab) and same(top_k=2 ** 31 - 1)
    assert same(top_p=1.0) and same(top_p=7.0) and same(top_p=np.nan)
    assert same(min_p=0.0) and same(min_p=-1.0) and same(min_p=np.nan) and same(temperature=1.0)
    first = l.argmax(1)
    takes = lambda **kw: np.array_equal(
        _run(l, u, **{k: np.full(rows, v) for k, v in kw.items()})[0], first)
    assert takes(temperature=0.0) and takes(temperature=-1.0) and takes(temperature=np.nan)
    assert takes(top_k=1) and takes(top_p=0.0) and takes(top_p=-2.0) and takes(min_p=1.0)
    assert takes(min_p=9.0) and takes(temperature=1e-38)
    assert np.array_equal(_run(l, np.full(rows, -1.0))[0], first)
    last, _ = _run(l, np.full(rows, 1 - 2.0 ** -24))
    for v in (1.0, 3.0, np.nan, np.inf):
        assert np.array_equal(_run(l, np.full(rows, v))[0], last)


def test_rows_do_not_meet(gpu):
    """A row's token is the same alone and in any batch, in any place and alignment."""
    import torch

    from deltafin_amd import sampling
    say("rows alone and together")
    torch.manual_seed(1)
    l = 2 * torch.randn(70, 10007, device="cuda")
    u = torch.rand(70, device="cuda")
    k = torch.randint(0, 300, (70,), device="cuda", dtype=torch.int32)
    p = torch.rand(70, device="cuda") * 0.5 + 0.5
    for dtype in (torch.float32, torch.bfloat16):
        x = l.to(dtype)
        whole = sampling.sample(x, u, top_k=k, top_p=p)
        for i in (0, 1, 33, 69):
            one = sampling.sample(x[i:i + 1].contiguous(), u[i:i + 1], top_k=k[i:i + 1],
                                  top_p=p[i:i + 1])
            assert one.item() == whole[i].item()


def test_draws_follow_the_weights(gpu):
    """A grid of u over one row hits each token as often as its weight says, to one step."""
    say("grid of u")
    rng = np.random.default_rng(8)
    vocab, n = 11, 4096
    l = rng.standard_normal(vocab).astype(np.float32)
    found, _ = _run(np.tile(l, (n, 1)), (np.arange(n) + 0.5) / n)
    w = np.exp(l.astype(np.float64))
    want = n * w / w.sum()
    assert np.all(np.abs(np.bincount(found, minlength=vocab) - want) <= 1 + 1e-6)


def test_graph_stream_and_workspace(gpu):
    import torch

    from deltafin_amd import sampling
    say("graph, stream, workspace")
    torch.manual_seed(2)
    l = torch.randn(12, 30001, device="cuda")
    u = torch.rand(12, device="cuda")
    p = torch.full((12,), 0.9, device="cuda")
    ws = torch.full((4 << 20,), 255, dtype=torch.uint8, device="cuda")
    want = sampling.sample(l, u, top_p=p)
    for _ in range(2):
        assert torch.equal(sampling.sample(l, u, top_p=p, workspace=ws), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = sampling.sample(l, u, top_p=p)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = sampling.sample(l, u, top_p=p)
    for _ in range(4):
        l.copy_(torch.randn(12, 30001, device="cuda"))
        u.copy_(torch.rand(12, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, sampling.sample(l, u, top_p=p))


def test_torch_interface_refusals(gpu):
    import torch

    from deltafin_amd import sampling
    l, u = torch.zeros(3, 50, device="cuda"), torch.zeros(3, device="cuda")
    for bad in (lambda: sampling.sample(l.half(), u), lambda: sampling.sample(l.t(), u),
                lambda: sampling.sample(l, u[:2]), lambda: sampling.sample(l, u.double()),
                lambda: sampling.sample(l, u, top_k=u), lambda: sampling.sample(l, u, top_p=u[:1]),
                lambda: sampling.sample(l, u, out=u), lambda: sampling.sample(l, u, workspace=u)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(Exception, match="must be 1.."):
        sampling.sample(l[:0], u[:0])
