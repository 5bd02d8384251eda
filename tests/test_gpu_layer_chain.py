"""A feed-forward layer, the head and the sampler as a decoder runs them: norm, gated block,
down projection onto the residual, head over the last positions, a token per row; at a
prompt's length, at a draft's and at one position, against the float64 oracles.  And one
training step of the layer by its gradient."""
import numpy as np
import pytest

from oracle import dense as D
from oracle.sampling import sample_row

pytestmark = pytest.mark.gpu


def _layer(rng, kind, hidden, inter, vocab):
    import torch

    def matrix(rows, cols):
        if kind == "int8":
            q = rng.integers(-127, 128, (rows, cols)).astype(np.int8)
            s = np.full(rows, 1 / (73 * np.sqrt(cols)), np.float32)
            return torch.from_numpy(q).cuda(), torch.from_numpy(s).cuda(), q * s[:, None]
        v = D.bf16_round((rng.standard_normal((rows, cols)) / np.sqrt(cols)).astype(np.float32))
        return torch.from_numpy(v).cuda().bfloat16(), None, v

    return [matrix(inter, hidden), matrix(inter, hidden), matrix(hidden, inter),
            matrix(vocab, hidden)], (1 + 0.1 * rng.standard_normal(hidden)).astype(np.float32)


@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("positions", [1, 5, 40, 300])
def test_layer_head_and_tokens(gpu, kind, positions):
    import torch

    from deltafin_amd import dense, sampling, spine
    rng = np.random.default_rng(positions)
    hidden, inter, vocab = 264, 520, 4111
    (wg, wu, wd, head), norm = _layer(rng, kind, hidden, inter, vocab)
    x = rng.standard_normal((positions, hidden)).astype(np.float32)
    print(f"[gpu-case] layer {kind} {positions}", flush=True)
    dx = torch.from_numpy(x).cuda()
    n = spine.rms_norm(dx, torch.from_numpy(norm).cuda())
    h = dense.gated_ffn(wg[0], wu[0], n, "situ", gate_scales=wg[1], up_scales=wu[1])
    y = dense.linear(wd[0], h, residual=dx, row_scales=wd[1])
    last = min(positions, 4)
    logits = dense.linear(head[0], y[-last:], row_scales=head[1])
    u = torch.rand(last, device="cuda")
    kw = dict(top_k=torch.full((last,), 50, dtype=torch.int32, device="cuda"),
              top_p=torch.full((last,), 0.9, device="cuda"))
    tokens = sampling.sample(logits, u, **kw)
    torch.cuda.synchronize()
    x64 = x.astype(np.float64)
    n64 = norm * x64 / np.sqrt((x64 ** 2).mean(1, keepdims=True) + 1e-5)
    f, _, _ = D.gate("situ", n64 @ wg[2].T.astype(np.float64), n64 @ wu[2].T.astype(np.float64))
    y64 = f @ wd[2].T.astype(np.float64) + x64
    want = y64[-last:] @ head[2].T.astype(np.float64)
    # four sums of at most 520 terms one behind the other, each off by at most
    # (terms + 8) half steps of its magnitudes, which are under 30 here for outputs of order 1
    tol = 4 * (520 + 8) * 30 * D.F32_HALF_STEP
    assert np.abs(logits.cpu().numpy() - want).max() <= tol
    read = logits.cpu().numpy()
    for i in range(last):
        token, margin = sample_row(read[i], float(u[i]), top_k=50, top_p=float(np.float32(0.9)))
        assert margin < 2.0 ** -36 or tokens[i].item() == token


def test_a_step_moves_the_loss_as_the_gradient_says(gpu):
    """One step of the gated block against a fixed direction: the loss moves by what the
    gradient says, to the second order of the step."""
    import torch

    from deltafin_amd import dense
    torch.manual_seed(1)
    P, R, H = 300, 136, 200
    wg, wu = ((torch.randn(R, H, device="cuda") / 14).bfloat16() for _ in range(2))
    x, d = torch.randn(P, H, device="cuda"), torch.randn(P, R, device="cuda")
    loss = lambda a, b: (dense.gated_ffn(a, b, x).double() * d.double()).sum().item()
    h, g, u = dense.gated_ffn(wg, wu, x, keep=True)
    _, d_gate, d_up = dense.gated_ffn_backward(wg, wu, x, g, u, d)
    base = loss(wg, wu)
    for rate in (2.0 ** -10, 2.0 ** -12):
        a = (wg.float() - rate * d_gate).bfloat16()
        b = (wu.float() - rate * d_up).bfloat16()
        # what the rounded weights really moved by
        da, db = a.double() - wg.double(), b.double() - wu.double()
        want = (da * d_gate.double()).sum().item() + (db * d_up.double()).sum().item()
        # second derivatives of silu(g) u are under 1.2 (|u| + 1), at the larger of g and u
        # on the way: projections of the step squared
        pa, pb = x.double() @ da.t(), x.double() @ db.t()
        far = 2 + g.double().abs() + u.double().abs() + pa.abs() + pb.abs()
        second = (1.2 * d.double().abs() * (pa.abs() + pb.abs()) ** 2 * far).sum().item()
        rounding = 2.0 ** -18 * d.abs().sum().item()
        assert abs(loss(a, b) - base - want) <= second + rounding
