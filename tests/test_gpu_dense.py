"""Dense layers on the GPU against the float64 oracle (oracle/dense.py), under bounds
derived there from the number of roundings; products of small integers, whose sums are
exact, bit for bit at the large sizes."""
import numpy as np
import pytest

from oracle import dense as D

pytestmark = pytest.mark.gpu


def say(msg):
    print(f"[gpu-case] {msg}", flush=True)


def _dev(v, dtype):
    """The device tensor of fp32 values and the values that it holds."""
    import torch
    t = torch.from_numpy(np.ascontiguousarray(v, np.float32)).to(dtype)
    return t.cuda(), t.float().numpy()


def _dt(name):
    import torch
    return {"f32": torch.float32, "bf16": torch.bfloat16}[name]


def _matrix(rng, kind, rows, cols):
    """(device matrix, device scales or None, its values, scales)"""
    import torch
    if kind == "int8":
        q = rng.integers(-127, 128, (rows, cols)).astype(np.int8)
        s = (rng.uniform(0.5, 1.5, rows) / (73 * np.sqrt(cols))).astype(np.float32)
        return torch.from_numpy(q).cuda(), torch.from_numpy(s).cuda(), q, s
    t, v = _dev(rng.standard_normal((rows, cols)) / np.sqrt(cols), torch.bfloat16)
    return t, None, v, None


def _close(found, want, bound, dtype, tag):
    found = found.float().cpu().numpy().astype(np.float64)
    assert found.shape == want.shape, tag
    half = D.BF16_HALF_STEP if dtype == "bf16" else D.F32_HALF_STEP
    tol = bound + half * (np.abs(want) + bound) + 2.0 ** -148
    err = np.abs(found - want)
    assert np.all(np.isfinite(found)), f"{tag}: not finite"
    worst = np.unravel_index(np.argmax(err - tol), err.shape)
    assert np.all(err <= tol), f"{tag}: {err[worst]:.3e} > {tol[worst]:.3e} at {worst}"


SHAPES = [(1, 7, 5), (1, 64, 128), (3, 130, 72), (17, 1, 64), (64, 257, 600), (65, 16, 1),
          (129, 136, 344), (200, 513, 33), (300, 96, 520),
          (520, 96, 520), (530, 257, 72)]


@pytest.mark.parametrize("positions,rows,cols", SHAPES)
@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("x_dt,out_dt", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32")])
def test_linear(gpu, positions, rows, cols, kind, x_dt, out_dt):
    import torch

    from deltafin_amd import dense
    rng = np.random.default_rng(positions * 131 + rows * 7 + cols)
    w, s, wv, sv = _matrix(rng, kind, rows, cols)
    x, xv = _dev(rng.standard_normal((positions, cols)), _dt(x_dt))
    b = rng.standard_normal(rows).astype(np.float32)
    r, rv = _dev(rng.standard_normal((positions, rows)), _dt(out_dt))
    for act, bias, res in ((None, False, False), ("silu", True, False), ("gelu", True, True),
                           (None, False, True)):
        say(f"linear {positions}x{rows}x{cols} {kind} {x_dt}->{out_dt} {act} {bias} {res}")
        out = dense.linear(w, x, bias=torch.from_numpy(b).cuda() if bias else None, activation=act,
                           residual=r if res else None, row_scales=s, out_dtype=_dt(out_dt))
        torch.cuda.synchronize()
        want, bound = D.linear(wv, xv, b if bias else None, act, rv if res else None, sv)
        _close(out, want, bound, out_dt, f"{act} {bias} {res}")


def _ints(rng, shape, lo, hi):
    return rng.integers(lo, hi + 1, shape).astype(np.float32)


@pytest.mark.parametrize("positions,rows,cols", [(1, 7168, 2048), (9, 896, 7168), (48, 3584, 7168),
                                                 (100, 7168, 6144), (517, 2050, 7168),
                                                 (1024, 7168, 2048), (2048, 7168, 208),
                                                 (2100, 6144, 1003)])
@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("x_dt", ["f32", "bf16"])
def test_linear_integers_are_exact(gpu, positions, rows, cols, kind, x_dt):
    """Integers whose magnitudes' sum is under 2^24, so that every partial sum in every order
    is exact; fp32 rows hold more bits than one BF16 term."""
    import torch

    from deltafin_amd import dense
    rng = np.random.default_rng(positions + rows + cols)
    say(f"exact linear {positions}x{rows}x{cols} {kind} {x_dt}")
    most_w, most_x = (1, 2047) if x_dt == "f32" else (8, 255)
    assert cols * most_w * most_x < 2 ** 24
    wv = _ints(rng, (rows, cols), -most_w, most_w)
    xv = _ints(rng, (positions, cols), -most_x, most_x)
    w = torch.from_numpy(wv).cuda().to(torch.int8 if kind == "int8" else torch.bfloat16)
    s = torch.full((rows,), 0.5, device="cuda") if kind == "int8" else None
    x = torch.from_numpy(xv).cuda().to(_dt(x_dt))
    res = torch.from_numpy(_ints(rng, (positions, rows), -3, 3)).cuda()
    out = dense.linear(w, x, residual=res, row_scales=s, out_dtype=torch.float32)
    torch.cuda.synchronize()
    want = x.double() @ w.double().t() * (0.5 if kind == "int8" else 1.0) + res.double()
    assert torch.equal(out.double(), want)


@pytest.mark.parametrize("x_dt", ["f32", "bf16"])
@pytest.mark.parametrize("kind", ["bf16", "int8"])
def test_linear_every_alignment_of_views(gpu, kind, x_dt):
    """Operands that start anywhere in a buffer, and what lies around the output."""
    import torch

    from deltafin_amd import dense
    rng = np.random.default_rng(11)
    rows, cols, positions = 72, 160, 37
    w0, s, wv, sv = _matrix(rng, kind, rows, cols)
    x0, xv = _dev(rng.standard_normal((positions, cols)), _dt(x_dt))
    want, bound = D.linear(wv, xv, scales=sv)
    for off in (1, 2, 3, 8):
        say(f"view offset {off}")
        w = torch.zeros(rows * cols + off, dtype=w0.dtype, device="cuda")[off:].view(rows, cols)
        w.copy_(w0)
        x = torch.zeros(positions * cols + off, dtype=x0.dtype, device="cuda")[off:].view(
            positions, cols)
        x.copy_(x0)
        buf = torch.full((positions * rows + 2 * off,), 7.0, dtype=x0.dtype, device="cuda")
        out = dense.linear(w, x, row_scales=s, out=buf[off:off + positions * rows].view(
            positions, rows))
        torch.cuda.synchronize()
        _close(out, want, bound, x_dt, f"offset {off}")
        assert (buf[:off] == 7).all() and (buf[off + positions * rows:] == 7).all()


def test_linear_residual_in_place_and_single_row(gpu):
    import torch

    from deltafin_amd import dense
    rng = np.random.default_rng(5)
    w, _, wv, _ = _matrix(rng, "bf16", 256, 512)
    for positions in (1, 40, 300):
        say(f"in place {positions}")
        x, xv = _dev(rng.standard_normal((positions, 512)), torch.bfloat16)
        r, rv = _dev(rng.standard_normal((positions, 256)), torch.bfloat16)
        want, bound = D.linear(wv, xv, residual=rv)
        out = dense.linear(w, x, residual=r, out=r)
        torch.cuda.synchronize()
        assert out.data_ptr() == r.data_ptr()
        _close(out, want, bound, "bf16", f"in place {positions}")
    x, xv = _dev(rng.standard_normal(512), torch.float32)
    out = dense.linear(w, x)
    torch.cuda.synchronize()
    want, bound = D.linear(wv, xv[None])
    _close(out, want, bound, "f32", "one row")


@pytest.mark.parametrize("positions", [1, 20, 200])
def test_linear_fp32_range(gpu, positions):
    """Rows near both ends of fp32's range keep its precision beside ordinary ones; zeros
    stay zeros."""
    import torch

    from deltafin_amd import dense
    rng = np.random.default_rng(7)
    w, _, wv, _ = _matrix(rng, "bf16", 48, 264)
    xv = rng.standard_normal((positions, 264))
    scale = np.array([2.0 ** e for e in (0, -120, 118, -126, 60)])[np.arange(positions) % 5]
    xv = (xv * scale[:, None]).astype(np.float32)
    xv[positions // 2] = 0
    out = dense.linear(w, torch.from_numpy(xv).cuda())
    torch.cuda.synchronize()
    want, bound = D.linear(wv, xv)
    # results under 2^-126 are multiples of 2^-149
    _close(out, want, bound + 2.0 ** -149, "f32", "range")
    assert (out[positions // 2] == 0).all()


@pytest.mark.parametrize("x_dt", ["f32", "bf16"])
@pytest.mark.parametrize("positions", [3, 24, 150])
def test_linear_non_finite_rows_stay_their_own(gpu, x_dt, positions):
    """An infinity or NaN in one activation row reaches that row alone, as IEEE sums do."""
    import torch

    from deltafin_amd import dense
    rng = np.random.default_rng(9)
    w, _, wv, _ = _matrix(rng, "bf16", 70, 128)
    _, xv = _dev(rng.standard_normal((positions, 128)), _dt(x_dt))
    clean, bound = D.linear(wv, xv)
    bad = xv.copy()
    bad[0, 3] = np.inf
    bad[1, 100] = np.nan
    out = dense.linear(w, torch.from_numpy(bad).cuda().to(_dt(x_dt)))
    torch.cuda.synchronize()
    f = out.float().cpu().numpy()
    with np.errstate(invalid="ignore"):
        want = wv[:, 3] * np.inf
    assert np.array_equal(f[0], want, equal_nan=True)
    assert np.isnan(f[1]).all()
    _close(out[2:], clean[2:], bound[2:], x_dt, "other rows")


GATED = [(1, 16, 8), (1, 40, 264), (5, 33, 70), (70, 130, 128), (131, 200, 328), (300, 64, 65),
         (515, 48, 264)]


@pytest.mark.parametrize("positions,rows,cols", GATED)
@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("x_dt,out_dt", [("f32", "f32"), ("bf16", "bf16"), ("f32", "bf16")])
@pytest.mark.parametrize("act", ["silu", "situ"])
def test_gated(gpu, positions, rows, cols, kind, x_dt, out_dt, act):
    import torch

    from deltafin_amd import dense
    rng = np.random.default_rng(positions * 31 + rows + cols)
    wg, gs, wgv, gsv = _matrix(rng, kind, rows, cols)
    wu, us, wuv, usv = _matrix(rng, kind, rows, cols)
    x, xv = _dev(2 * rng.standard_normal((positions, cols)), _dt(x_dt))
    (h, g, u), bounds = D.gated(wgv, wuv, xv, act, gsv, usv)
    say(f"gated {positions}x{rows}x{cols} {kind} {x_dt}->{out_dt} {act}")
    kept = dense.gated_ffn(wg, wu, x, act, keep=True, gate_scales=gs, up_scales=us,
                           out_dtype=_dt(out_dt))
    alone = dense.gated_ffn(wg, wu, x, act, gate_scales=gs, up_scales=us, out_dtype=_dt(out_dt))
    torch.cuda.synchronize()
    for f, want, bound, name in zip(kept, (h, g, u), bounds, "hgu"):
        _close(f, want, bound, out_dt, name)
    _close(alone, h, bounds[0], out_dt, "h alone")


@pytest.mark.parametrize("positions,rows,cols", [(1, 6144, 7168), (16, 2048, 7168),
                                                 (700, 2048, 7168), (1030, 1003, 2050)])
@pytest.mark.parametrize("x_dt", ["f32", "bf16"])
def test_gated_integers_are_exact(gpu, positions, rows, cols, x_dt):
    import torch

    from deltafin_amd import dense
    rng = np.random.default_rng(positions + rows)
    say(f"exact gated {positions}x{rows}x{cols} {x_dt}")
    wg, wu = (torch.from_numpy(_ints(rng, (rows, cols), -8, 8)).cuda().to(torch.bfloat16)
              for _ in range(2))
    x = torch.from_numpy(_ints(rng, (positions, cols), -255, 255)).cuda().to(_dt(x_dt))
    _, g, u = dense.gated_ffn(wg, wu, x, "silu", keep=True, out_dtype=torch.float32)
    torch.cuda.synchronize()
    assert torch.equal(g.double(), x.double() @ wg.double().t())
    assert torch.equal(u.double(), x.double() @ wu.double().t())


@pytest.mark.parametrize("positions,rows,cols", [(1, 8, 16), (16, 33, 70), (130, 130, 72),
                                                 (300, 64, 65), (520, 257, 264)])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("act", ["silu", "situ"])
def test_gated_backward(gpu, positions, rows, cols, dt, act):
    import torch

    from deltafin_amd import dense
    rng = np.random.default_rng(positions + rows * 5 + cols)
    wg, _, wgv, _ = _matrix(rng, "bf16", rows, cols)
    wu, _, wuv, _ = _matrix(rng, "bf16", rows, cols)
    x, xv = _dev(rng.standard_normal((positions, cols)), _dt(dt))
    g, gv = _dev(2 * rng.standard_normal((positions, rows)), _dt(dt))
    u, uv = _dev(2 * rng.standard_normal((positions, rows)), _dt(dt))
    d, dv = _dev(rng.standard_normal((positions, rows)), _dt(dt))
    say(f"backward {positions}x{rows}x{cols} {dt} {act}")
    found = dense.gated_ffn_backward(wg, wu, x, g, u, d, act)
    torch.cuda.synchronize()
    wants, bounds = D.gated_grad(wgv, wuv, xv, gv, uv, dv, act, dt)
    for f, want, bound, name in zip(found, wants, bounds, ("d_x", "d_gate", "d_up")):
        _close(f, want, bound, dt, name)


@pytest.mark.parametrize("positions,rows,cols", [(4096, 264, 2050), (1000, 2048, 1536),
                                                 (517, 1003, 2050), (2048, 136, 7168),
                                                 (200, 1024, 7168)])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_gated_backward_integers_are_exact(gpu, positions, rows, cols, dt):
    """g = 0 makes SiLU's dg = grad u / 2 and du = 0, g = 100 makes dg = grad u and du =
    100 grad to their last bit (the sigmoid is 1 / 2 and 1); small integers then make every
    sum exact."""
    import torch

    from deltafin_amd import dense
    rng = np.random.default_rng(rows)
    say(f"exact backward {positions}x{rows}x{cols} {dt}")
    dtype = _dt(dt)
    on = lambda v: torch.from_numpy(v.astype(np.float32)).cuda()
    wg, wu = (on(_ints(rng, (rows, cols), -4, 4)).bfloat16() for _ in range(2))
    x = on(_ints(rng, (positions, cols), -4, 4)).to(dtype)
    g = on(100.0 * rng.integers(0, 2, (positions, rows))).to(dtype)
    u = on(_ints(rng, (positions, rows), -4, 4)).to(dtype)
    d = on(_ints(rng, (positions, rows), -1, 1)).to(dtype)
    d_x, d_gate, d_up = dense.gated_ffn_backward(wg, wu, x, g, u, d, "silu")
    torch.cuda.synchronize()
    sig = torch.where(g > 0, 1.0, 0.5).double()
    # gate 100: sig (1 + g (1 - sig)) is 1 exactly, since 1 - sig rounds to zero
    dg, du = d.double() * u.double() * sig, d.double() * g.double() * sig
    for f, want in ((d_x, dg @ wg.double() + du @ wu.double()), (d_gate, dg.t() @ x.double()),
                    (d_up, du.t() @ x.double())):
        assert want.abs().max() < 2 ** 24
        assert torch.equal(f, want.to(dtype))


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("positions", [37, 128])
def test_gated_backward_every_alignment_of_views(gpu, positions, dt):
    """Any of the operands copied, the others in place: sums of small integers, bit for bit
    (as above)."""
    import torch

    from deltafin_amd import dense
    rng = np.random.default_rng(positions)
    rows, cols = 72, 160
    dtype = _dt(dt)

    def at(v, dtype, off):
        flat = torch.full((v.size + off + 8,), float("nan"), dtype=dtype, device="cuda")
        view = flat[off:off + v.size].view(v.shape)
        view.copy_(torch.from_numpy(v.astype(np.float32)))
        return view

    wg, wu = (_ints(rng, (rows, cols), -4, 4) for _ in range(2))
    x = _ints(rng, (positions, cols), -4, 4)
    g = 100.0 * rng.integers(0, 2, (positions, rows))
    u = _ints(rng, (positions, rows), -4, 4)
    d = _ints(rng, (positions, rows), -1, 1)
    sig = np.where(g > 0, 1.0, 0.5)
    dg, du = d * u * sig, d * g * sig
    wants = [torch.from_numpy(np.asarray(v, np.float64)).to(dtype).cuda()
             for v in (dg @ wg + du @ wu, dg.T @ x, du.T @ x)]
    for offs in ((0, 0, 0, 0), (1, 0, 0, 0), (0, 1, 0, 0), (0, 0, 1, 0), (3, 5, 0, 1),
                 (0, 8, 2, 0), (1, 1, 1, 1)):
        say(f"backward views {offs} {dt}")
        og, ou, ox, oa = offs
        found = dense.gated_ffn_backward(
            at(wg, torch.bfloat16, og), at(wu, torch.bfloat16, ou), at(x, dtype, ox),
            at(g, dtype, oa), at(u, dtype, 0), at(d, dtype, oa), "silu")
        torch.cuda.synchronize()
        for f, want, name in zip(found, wants, ("d_x", "d_gate", "d_up")):
            assert torch.equal(f, want), (offs, name)


@pytest.mark.parametrize("act", ["silu", "situ"])
def test_gated_backward_against_differences(gpu, act):
    """Differences of the kernel's own forward pass: a step of 2^-6 along a direction moves
    the loss by the gradient's share up to the step's cube and the sums' roundings."""
    import torch

    from deltafin_amd import dense
    torch.manual_seed(2)
    P, R, H = 40, 48, 64
    wg, wu = ((torch.randn(R, H, device="cuda") / 8).bfloat16() for _ in range(2))
    x, d = torch.randn(P, H, device="cuda"), torch.randn(P, R, device="cuda")
    _, g, u = dense.gated_ffn(wg, wu, x, act, keep=True)
    d_x, _, _ = dense.gated_ffn_backward(wg, wu, x, g, u, d, act)
    v = torch.randn(P, H, device="cuda")
    step = 2.0 ** -6
    loss = lambda at: (dense.gated_ffn(wg, wu, at, act).double() * d.double()).sum().item()
    diff = (loss(x + step * v) - loss(x - step * v)) / (2 * step)
    want = (d_x.double() * v.double()).sum().item()
    # third derivatives of f are under 2 per (|g| + |u| + 1); projections of v are of
    # order 1: the cubic term is at most 2 * step^2 / 6 * sum |d| (|Wv|^3 (|g| + |u| + 1))
    pg, pu = v.double() @ wg.double().t(), v.double() @ wu.double().t()
    cubic = 2 * step ** 2 / 6 * (d.double().abs() * (pg.abs() + pu.abs()) ** 3
                                 * (g.double().abs() + u.double().abs() + 1)).sum().item()
    rounding = 2 ** -18 * (d.abs().sum().item()) / step
    assert abs(diff - want) <= cubic + rounding, (diff, want, cubic, rounding)


def test_workspace_contents_do_not_matter(gpu):
    """A workspace full of NaN patterns, one that another call has used, and one larger than
    needed give the same bits."""
    import torch

    from deltafin_amd import dense
    torch.manual_seed(4)
    w = torch.randn(136, 333, device="cuda").bfloat16()
    x = torch.randn(70, 333, device="cuda")
    want = dense.linear(w, x)
    ws = torch.full((8 << 20,), 255, dtype=torch.uint8, device="cuda")
    for _ in range(2):
        assert torch.equal(dense.linear(w, x, workspace=ws), want)
    g = torch.randn(70, 136, device="cuda")
    first = dense.gated_ffn_backward(w, w, x, g, g, g)
    ws.fill_(255)
    for a, b in zip(dense.gated_ffn_backward(w, w, x, g, g, g, workspace=ws), first):
        assert torch.equal(a, b)
    with pytest.raises(Exception, match="workspace"):
        dense.linear(w, x, workspace=ws[:128])


def test_other_stream_and_graph(gpu):
    """A feed-forward layer with its gradient on a stream of its own, captured and replayed
    with new inputs between the replays, equal to eager calls."""
    import torch

    from deltafin_amd import dense
    torch.manual_seed(6)
    P, R, H = 150, 264, 512
    wg, wu = ((torch.randn(R, H, device="cuda") / 20).bfloat16() for _ in range(2))
    wd = (torch.randn(H, R, device="cuda") / 16).bfloat16()
    x = torch.randn(P, H, device="cuda")
    dh = torch.randn(P, R, device="cuda")

    def layer():
        h, g, u = dense.gated_ffn(wg, wu, x, "situ", keep=True)
        y = dense.linear(wd, h, residual=x)
        return (y, *dense.gated_ffn_backward(wg, wu, x, g, u, dh, "situ"))

    eager = layer()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = layer()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(eager, again))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer()
    for k in range(3):
        x.copy_(torch.randn(P, H, device="cuda"))
        dh.copy_(torch.randn(P, R, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        want = layer()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), k


def test_torch_interface_refusals(gpu):
    import torch

    from deltafin_amd import dense
    w = torch.zeros(16, 32, dtype=torch.bfloat16, device="cuda")
    q = torch.zeros(16, 32, dtype=torch.int8, device="cuda")
    x = torch.zeros(4, 32, device="cuda")
    bad = [
        lambda: dense.linear(w, x[:, :16]), lambda: dense.linear(w, x.half()),
        lambda: dense.linear(w.t(), x), lambda: dense.linear(w.float(), x),
        lambda: dense.linear(q, x), lambda: dense.linear(w, x, row_scales=x[0, :16]),
        lambda: dense.linear(w, x, bias=torch.zeros(15, device="cuda")),
        lambda: dense.linear(w, x, activation="relu"),
        lambda: dense.linear(w, x, residual=torch.zeros(4, 16, device="cuda").bfloat16()),
        lambda: dense.linear(w, x, out=torch.zeros(4, 17, device="cuda")),
        lambda: dense.linear(w, x, out_dtype=torch.float16),
        lambda: dense.linear(w, x, workspace=x),
        lambda: dense.gated_ffn(w, q, x), lambda: dense.gated_ffn(w, w[:8], x),
        lambda: dense.gated_ffn(w, w, x, "gelu"), lambda: dense.gated_ffn(w, w, x, True),
        lambda: dense.gated_ffn_backward(w, w, x, x, x, x),
        lambda: dense.gated_ffn_backward(q, q, x, x[:, :16], x[:, :16], x[:, :16]),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            raise AssertionError(i)
    with pytest.raises(Exception, match="1..1048576"):
        dense.linear(w, torch.zeros(0, 32, device="cuda"))
