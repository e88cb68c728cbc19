"""The LM head's cross entropy and its gradient (``cid_engine.lm_head_cross_entropy``)
against the formula in 64 bits, from the same 16-bit inputs.

Tolerances, element by element, from the roundings that the operator makes:

* a logit z = h . w is a float32 sum on the tensor cores: at most
  (H / 16 + 16) steps of 2^-22 of sum |h w| (each 16-wide step may truncate);
  that bounds log-sum-exp and, twice, the loss, next to 2^-21 of the value for
  exp, log and the final subtraction;
* d = a exp(z - lse) - b [label] is rounded to 16 bits (half a step u =
  finfo.eps / 2 of each element) after the logits' error moved it by a
  relative 2 dz + 2^-20: |dh| is off by at most (u + 2 dz + 2^-20) (|d| |W|)
  with |d| <= |a| p + |b| [label], plus u |dh| for its own rounding and the
  float32 sums' (V / 16 + 80) 2^-22 of |d| |W|; dW likewise over the rows;
* fp16 adds half its smallest subnormal (2^-25) to an output, and 2^-25 over
  the scale of d (at least 2^12 over the largest coefficient) times |W|'s or
  |h|'s sum to a gradient.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


@pytest.fixture(scope="module", autouse=True)
def _engine():
    import cid_engine  # noqa: F401

    assert torch.cuda.is_available()
    yield
    torch.cuda.empty_cache()


def _inputs(rows, vocab, hidden, dtype, keep="half", seed=0):
    dev = torch.device("cuda", 0)
    g = torch.Generator(device=dev).manual_seed(seed + rows * 7 + vocab * 3 + hidden)
    h = torch.randn(rows, hidden, generator=g, device=dev).to(dtype)
    w = (torch.randn(vocab, hidden, generator=g, device=dev) * (2.0 / hidden**0.5)).to(dtype)
    y = torch.randint(0, vocab, (rows,), generator=g, device=dev)
    drop = {
        "all": torch.zeros(rows, dtype=torch.bool, device=dev),
        "none": torch.ones(rows, dtype=torch.bool, device=dev),
        "half": torch.rand(rows, generator=g, device=dev) < 0.5,
        "last": torch.arange(rows, device=dev) != rows - 1,
        "first": torch.arange(rows, device=dev) != 0,
    }[keep]
    y[drop] = -100
    gl = torch.rand(rows, generator=g, device=dev) + 0.25
    ge = torch.randn(rows, generator=g, device=dev) * 0.1
    return y, h, w, gl, ge


def _exact(y, h, w, gl, ge):
    """Outputs and gradients in 64 bits, and the sums the tolerances need."""
    keep = y >= 0
    hd = torch.where(keep[:, None], h.double(), 0.0)
    wd = w.double()
    z = hd @ wd.T
    lse = torch.logsumexp(z, 1)
    at = torch.where(keep, y, 0)
    one = torch.zeros_like(z).scatter_(1, at[:, None], 1.0)
    loss = lse - (z * one).sum(1)
    p = torch.exp(z - lse[:, None])
    a, b = (gl + ge).double() * keep, gl.double() * keep
    d = a[:, None] * p - b[:, None] * one
    dabs = a.abs()[:, None] * p + b.abs()[:, None] * one
    H, V, N = h.shape[1], w.shape[0], h.shape[0]
    dz = (H / 16 + 16) * 2.0**-22 * (hd.abs() @ wd.abs().T).amax(1)  # per row
    u = torch.finfo(h.dtype).eps / 2
    rel = u + 2 * dz[:, None] + 2.0**-20
    sub = 2.0**-25 if h.dtype == FP16 else 0.0
    dsub = sub * float(torch.maximum(a.abs(), b.abs()).max()) * 2.0**-12 if N else 0.0
    top_h, top_w = hd.abs(), wd.abs()
    dh, dw = d @ wd, d.T @ hd
    tol_dh = ((rel * dabs) @ top_w + (V / 16 + 80) * 2.0**-22 * (dabs @ top_w) + u * dh.abs()
              + sub + dsub * top_w.sum(0))
    tol_dw = ((rel * dabs).T @ top_h + (N / 16 + 80) * 2.0**-22 * (dabs.T @ top_h)
              + u * dw.abs() + sub + dsub * top_h.sum(0))
    loss, lse = torch.where(keep, loss, 0.0), torch.where(keep, lse, 0.0)
    tol = dz + 2.0**-21 * (lse.abs() + (z * one).sum(1).abs() + 1)
    return loss, lse, dh, dw, 2 * tol, tol, tol_dh, tol_dw


def _within(name, got, want, tol):
    off = (got.double() - want).abs()
    bad = ~(off <= tol * 1.001 + 1e-30)
    assert not bool(bad.any()), (
        f"{name}: {int(bad.sum())} of {bad.numel()} outside, worst {float((off / (tol + 1e-30)).max()):.3g} "
        f"of the tolerance")


def _step(y, h, w, gl, ge):
    import cid_engine

    h, w = h.detach().requires_grad_(), w.detach().requires_grad_()
    loss, lse = cid_engine.lm_head_cross_entropy(y, h, w)
    dh, dw = torch.autograd.grad((loss, lse), (h, w), grad_outputs=(gl, ge))
    return loss.detach(), lse.detach(), dh, dw


def _check(y, h, w, gl, ge):
    import cid_engine

    cid_engine.device_status(0, reset=True)
    got = _step(y, h, w, gl, ge)
    assert cid_engine.device_status(0) == 0
    loss, lse, dh, dw, t_loss, t_lse, t_dh, t_dw = _exact(y, h, w, gl, ge)
    _within("loss", got[0], loss, t_loss)
    _within("log_sum_exp", got[1], lse, t_lse)
    _within("grad_hidden", got[2], dh, t_dh)
    _within("grad_weight", got[3], dw, t_dw)
    return got


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("rows,vocab,hidden", [
    (1, 1, 8),          # one token: loss 0
    (1, 7, 8),
    (2, 256, 64),
    (17, 257, 72),      # one column past a tile, a K tail
    (130, 1000, 136),   # one row past two row blocks
    (256, 513, 264),    # hidden one vector past a column tile
    (300, 5000, 1000),
    (700, 4099, 520),   # several row blocks and K slices of dW
])
def test_loss_and_gradients(rows, vocab, hidden, dtype) -> None:
    _check(*_inputs(rows, vocab, hidden, dtype, keep="half" if rows > 2 else "all"))


@pytest.mark.parametrize("keep", ["all", "none", "first", "last"])
@pytest.mark.parametrize("rows", [1, 16, 129, 260])
def test_kept_rows(rows, keep) -> None:
    """Rows without labels in any pattern, all of them among the patterns: their
    outputs and gradients are exactly zero."""
    y, h, w, gl, ge = _inputs(rows, 600, 64, BF16, keep)
    loss, lse, dh, dw = _check(y, h, w, gl, ge)
    out = y < 0
    assert not bool(loss[out].any()) and not bool(lse[out].any()) and not bool(dh[out].any())
    if keep == "none":
        assert not bool(dw.any())


@pytest.mark.parametrize("rows,vocab,hidden", [
    (9000, 20011, 64), (33000, 9001, 16), (40, 70001, 128), (3000, 12000, 256)])
def test_pieces_of_the_vocabulary(rows, vocab, hidden) -> None:
    """Sizes at which the backward takes several pieces (9000 rows: 14336 columns
    and a short piece; 33000: the least, 4096) or splits the sum over the
    vocabulary."""
    _check(*_inputs(rows, vocab, hidden, BF16))


def test_large_and_small_coefficients_in_fp16() -> None:
    """Loss scales of 65536 and weights of 1e-6: fp16's range is not left inside."""
    y, h, w, gl, ge = _inputs(100, 3000, 64, FP16)
    for s in (256.0, 1e-3):
        _check(y, h, w, gl * s, ge * s)
    _check(y, h, w * 0, gl, ge)


def test_ignored_rows_are_not_read() -> None:
    """NaN, infinities and huge values in rows without a label reach nothing."""
    y, h, w, gl, ge = _inputs(200, 900, 128, BF16)
    want = _step(y, h, w, gl, ge)
    bad = h.clone()
    rows = (y < 0).nonzero().flatten()
    bad[rows[0::3]] = float("nan")
    bad[rows[1::3]] = float("inf")
    bad[rows[2::3]] = -3e38
    gl2, ge2 = gl.clone(), ge.clone()
    gl2[rows], ge2[rows] = float("nan"), float("inf")
    for a, b in zip(_step(y, bad, w, gl2, ge2), want):
        assert torch.equal(a, b)


def test_labels_outside_the_vocabulary() -> None:
    import cid_engine

    y, h, w, gl, ge = _inputs(40, 500, 64, BF16, "all")
    without = y.clone()
    y[3], y[20], y[39] = 500, -1, 1 << 40
    without[[3, 20, 39]] = -100
    want = _step(without, h, w, gl, ge)
    cid_engine.device_status(0, reset=True)
    loss, lse, dh, dw = _step(y, h, w, gl, ge)
    assert cid_engine.device_status(0, reset=True) == cid_engine.STATUS_TOKEN_ID_OUT_OF_RANGE
    bad = torch.zeros(40, dtype=torch.bool, device=y.device)
    bad[[3, 20, 39]] = True
    for t in (loss, lse, dh):
        assert bool(t[bad].isnan().all())
    assert torch.equal(loss[~bad], want[0][~bad]) and torch.equal(dh[~bad], want[2][~bad])
    assert torch.equal(dw, want[3])


def test_ignore_index_is_any_value() -> None:
    import cid_engine

    y, h, w, _, _ = _inputs(64, 300, 64, BF16)
    other = torch.where(y < 0, torch.full_like(y, 7), torch.where(y == 7, torch.full_like(y, 8), y))
    base = torch.where(other == 7, torch.full_like(y, -100), other)
    a = cid_engine.lm_head_cross_entropy(other, h, w, ignore_index=7)
    b = cid_engine.lm_head_cross_entropy(base, h, w)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_not_finite_logits_stay_in_their_rows() -> None:
    """A NaN or infinite logit makes its own row's loss NaN and no other's."""
    import cid_engine

    y, h, w, _, _ = _inputs(150, 700, 64, BF16, "all")
    want, _ = cid_engine.lm_head_cross_entropy(y, h, w)
    h2 = h.clone()
    h2[5, 3], h2[77, 0], h2[149, 63] = float("nan"), float("inf"), -float("inf")
    loss, _ = cid_engine.lm_head_cross_entropy(y, h2, w)
    bad = torch.zeros(150, dtype=torch.bool, device=y.device)
    bad[[5, 77, 149]] = True
    assert bool(loss[bad].isnan().all()) and torch.equal(loss[~bad], want[~bad])


def test_shapes_strides_and_single_gradients() -> None:
    """Batched shapes, strided and offset views, a broadcast gradient, and one
    gradient at a time: the bits of the plain call."""
    import cid_engine

    y, h, w, gl, ge = _inputs(60, 400, 64, BF16)
    loss, lse, dh, dw = _step(y, h, w, gl, ge)
    wide = torch.zeros(60, 136, dtype=BF16, device=h.device)
    wide[:, 1:65] = h
    wt = w.T.contiguous().T
    yy = torch.stack([y, y], 1)[:, 0]
    l2, e2, dh2, dw2 = _step(yy, wide[:, 1:65], wt, gl, ge)
    assert torch.equal(loss, l2) and torch.equal(lse, e2)
    assert torch.equal(dh, dh2) and torch.equal(dw, dw2)
    flat = torch.empty(60 * 64 + 4, dtype=BF16, device=h.device)[4:].view(3, 20, 64)  # 8 bytes off
    flat.copy_(h.view(3, 20, 64))
    l3, e3, dh3, dw3 = _step(y.view(3, 20), flat, w, gl.view(3, 20), ge.view(3, 20))
    assert l3.shape == (3, 20) and torch.equal(l3.view(-1), loss)
    assert dh3.shape == (3, 20, 64) and torch.equal(dh3.view(60, 64), dh) and torch.equal(dw3, dw)
    hr = h.detach().requires_grad_()
    (only,) = torch.autograd.grad(cid_engine.lm_head_cross_entropy(y, hr, w)[0], hr, grad_outputs=gl)
    wr = w.detach().requires_grad_()
    (onlyw,) = torch.autograd.grad(cid_engine.lm_head_cross_entropy(y, h, wr)[0], wr, grad_outputs=gl)
    both = _step(y, h, w, gl, torch.zeros_like(ge))
    assert torch.equal(only, both[2]) and torch.equal(onlyw, both[3])
    hr = h.detach().requires_grad_()
    cid_engine.lm_head_cross_entropy(y, hr, w)[0].sum().backward()
    ones = _step(y, h, w, torch.ones_like(gl), torch.zeros_like(ge))
    assert torch.equal(hr.grad, ones[2])


def test_empty() -> None:
    import cid_engine

    w = torch.randn(50, 64, device="cuda").to(BF16).requires_grad_()
    h = torch.zeros(0, 64, device="cuda", dtype=BF16, requires_grad=True)
    loss, lse = cid_engine.lm_head_cross_entropy(torch.zeros(0, dtype=torch.long, device="cuda"), h, w)
    assert loss.shape == (0,) and lse.shape == (0,)
    loss.sum().backward()
    assert h.grad.shape == (0, 64) and not bool(w.grad.any())


def test_gradient_against_differences() -> None:
    """(L(x + t v) - L(x - t v)) / 2t for hidden and weight, in steps that the
    16-bit inputs hold exactly: inputs are multiples of 2^-5 below 2 (bf16
    holds 2^-6 there) and v is +-1.

    The difference's own error is t^2 / 6 of a third derivative, |L'''| <= 2 m^3
    for m the largest |logit change| per unit step, plus the loss's float32
    error over t; the gradient's is the sum of its elements' tolerances."""
    import cid_engine

    dev = torch.device("cuda", 0)
    g = torch.Generator(device=dev).manual_seed(3)
    N, V, H, t = 32, 96, 16, 2.0**-5
    h = (torch.randint(-31, 32, (N, H), generator=g, device=dev) * 2.0**-5).to(BF16)
    w = (torch.randint(-31, 32, (V, H), generator=g, device=dev) * 2.0**-5).to(BF16)
    y = torch.randint(0, V, (N,), generator=g, device=dev)
    y[::3] = -100
    n = int((y >= 0).sum())
    gl = torch.ones(N, device=dev)
    _, _, dh, dw = _step(y, h, w, gl, torch.zeros_like(gl))
    *_, tol_dh, tol_dw = _exact(y, h, w, gl, torch.zeros_like(gl))

    def total(a, b):
        return float(cid_engine.lm_head_cross_entropy(y, a, b)[0].double().sum())

    for grad, x, other, first, own in ((dh, h, w, True, tol_dh), (dw, w, h, False, tol_dw)):
        v = (torch.randint(0, 2, x.shape, generator=g, device=dev) * 2 - 1).to(BF16)
        up, down = (x + t * v), (x - t * v)
        assert torch.equal(up.double(), x.double() + t * v.double())
        d = (total(up, other) - total(down, other)) / (2 * t) if first else (
            total(other, up) - total(other, down)) / (2 * t)
        m = float((v.double() @ other.double().T).abs().max())
        tol = (n * (2 * m**3) * t**2 / 6 + n * 2 * 2.0**-20 * 8 / (2 * t)
               + float(own.sum()))
        assert abs(d - float((grad.double() * v.double()).sum())) <= tol
        assert tol < 3 * abs(d) + 20  # the tolerance says something


def test_repeated_calls_give_the_same_bits() -> None:
    x = _inputs(500, 9000, 256, BF16)
    first = _step(*x)
    for _ in range(3):
        for a, b in zip(_step(*x), first):
            assert torch.equal(a, b)


def test_graph_replays_with_other_labels() -> None:
    """The count of kept rows is read on the device: a captured step follows
    the labels, hidden states and weights it is replayed with."""
    import cid_engine

    y, h, w, gl, ge = _inputs(300, 2000, 128, BF16, "all")
    hr, wr = h.clone().requires_grad_(), w.clone().requires_grad_()
    ys = y.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            out = cid_engine.lm_head_cross_entropy(ys, hr, wr)
            torch.autograd.grad(out, (hr, wr), grad_outputs=(gl, ge))
    torch.cuda.current_stream().wait_stream(side)
    del out
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, lse = cid_engine.lm_head_cross_entropy(ys, hr, wr)
        dh, dw = torch.autograd.grad((loss, lse), (hr, wr), grad_outputs=(gl, ge))
    for keep in ("half", "none", "last", "all"):
        y2, h2, w2, _, _ = _inputs(300, 2000, 128, BF16, keep, seed=5)
        ys.copy_(y2)
        with torch.no_grad():
            hr.copy_(h2)
            wr.copy_(w2)
        graph.replay()
        for a, b in zip((loss, lse, dh, dw), _step(y2, h2, w2, gl, ge)):
            assert torch.equal(a, b)


def test_two_streams_at_once() -> None:
    x, x2 = _inputs(300, 3000, 128, BF16), _inputs(280, 5000, 192, FP16, seed=4)
    want, want2 = _step(*x), _step(*x2)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(4):
        with torch.cuda.stream(s1):
            a = _step(*x)
        with torch.cuda.stream(s2):
            b = _step(*x2)
        torch.cuda.synchronize()
        for got, ref in ((a, want), (b, want2)):
            for p, q in zip(got, ref):
                assert torch.equal(p, q)


def test_corruption_to_loss() -> None:
    """The training step these operators make together: masked positions of
    display_corrupt_from_random carry the loss, the others none, and the loss
    is that of the clean tokens there."""
    import cid_engine

    dev = torch.device("cuda", 0)
    g = torch.Generator(device=dev).manual_seed(1)
    B, L, V, H = 4, 96, 1200, 128
    ids = torch.randint(2, V, (B, L), generator=g, device=dev)
    corrupted, labels, masked, _ = cid_engine.display_corrupt_from_random(
        ids, torch.rand(B, generator=g, device=dev), torch.ones(B, L, dtype=torch.bool, device=dev),
        torch.rand(B, L, generator=g, device=dev), None, None, mask_token_id=0, eos_token_id=1,
        vocab_size=V, replacement_fraction=0.0)
    h = torch.randn(B, L, H, generator=g, device=dev).to(BF16)
    w = (torch.randn(V, H, generator=g, device=dev) * 0.2).to(BF16)
    gl = torch.rand(B * L, generator=g, device=dev)
    got = _step(labels, h, w, gl.view(B, L), torch.zeros(B, L, device=dev))
    flat = _exact(labels.view(-1), h.view(-1, H), w, gl, torch.zeros_like(gl))
    _within("loss", got[0].view(-1), flat[0], flat[4])
    _within("grad_hidden", got[2].view(-1, H), flat[2], flat[6])
    _within("grad_weight", got[3], flat[3], flat[7])
    assert torch.equal(got[0] != 0, labels >= 0)


def test_gradient_through_log_sum_exp_alone() -> None:
    """A penalty on the log-sum-exp: d = a p without the label's term."""
    import cid_engine

    y, h, w, _, ge = _inputs(90, 700, 128, BF16)
    hr, wr = h.detach().requires_grad_(), w.detach().requires_grad_()
    _, lse = cid_engine.lm_head_cross_entropy(y, hr, wr)
    dh, dw = torch.autograd.grad(lse, (hr, wr), grad_outputs=ge)
    exact = _exact(y, h, w, torch.zeros_like(ge), ge)
    _within("grad_hidden", dh, exact[2], exact[6])
    _within("grad_weight", dw, exact[3], exact[7])


def test_many_rows_few_labels() -> None:
    """Tiles and splits follow the kept rows, not the rows."""
    y, h, w, gl, ge = _inputs(2000, 4000, 192, BF16, "all")
    y[torch.arange(2000, device=y.device) % 167 != 3] = -100
    _check(y, h, w, gl, ge)


@pytest.mark.parametrize("keep", ["half", "last"])
def test_more_rows_than_packing_blocks(keep) -> None:
    """Of many rows a packing block takes several groups, one after the other."""
    _check(*_inputs(20011, 300, 64, BF16, keep))


def test_fp16_graphs_that_share_a_pool() -> None:
    """Two captured steps whose workspaces come from one pool, replayed in turn."""
    import cid_engine

    pool = torch.cuda.graph_pool_handle()
    steps = []
    for rows, vocab, hidden in ((300, 2000, 128), (60, 5000, 72)):
        y, h, w, gl, ge = _inputs(rows, vocab, hidden, FP16)
        hr, wr = h.clone().requires_grad_(), w.clone().requires_grad_()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            out = cid_engine.lm_head_cross_entropy(y, hr, wr)
            torch.autograd.grad(out, (hr, wr), grad_outputs=(gl, ge))
        torch.cuda.current_stream().wait_stream(side)
        del out
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            out = cid_engine.lm_head_cross_entropy(y, hr, wr)
            got = (*out, *torch.autograd.grad(out, (hr, wr), grad_outputs=(gl, ge)))
        steps.append((graph, got, _step(y, h, w, gl, ge), (y, hr, wr, gl, ge)))
    for _ in range(3):
        for graph, got, want, _ in steps:
            graph.replay()
            for a, b in zip(got, want):
                assert torch.equal(a, b)


@pytest.mark.parametrize("rows,tokens,hidden", [
    (64, 40, 72),     # two warps' tokens take every label, no more than are looked after
    (64, 32, 264),
    (40, 1, 520),     # one token's alone
    (200, 40, 136),   # more than are looked after
    (30, 17, 256),
])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_labels_of_few_tokens(rows, tokens, hidden, dtype) -> None:
    """dW's rows of the labels, where many of them are neighbours; a row without a
    gradient stands among them."""
    y, h, w, gl, ge = _inputs(rows, 2000, hidden, dtype, "all")
    y = 32 * 11 + y % tokens
    gl[rows // 2] = ge[rows // 2] = 0.0
    _check(y, h, w, gl, ge)
    y[rows // 4] = -100
    got = _check(y, h, w, gl, ge)
    for a, b in zip(_step(y, h, w, gl, ge), got):
        assert torch.equal(a, b)


# ---------------------------------------------------------------------------
# The label's element of d
# ---------------------------------------------------------------------------


def _steep(rows, vocab, hidden, dtype, labels, seed=0):
    """Inputs whose gradients are all but those of the labels: every logit but
    token 0's is about -24, so p is 1 at token 0 and below 1e-8 elsewhere, and
    token 0's weight row is zero.  ``labels`` are above 0."""
    dev = torch.device("cuda", 0)
    g = torch.Generator(device=dev).manual_seed(seed + rows + vocab)
    h = torch.randn(rows, hidden, generator=g, device=dev)
    w = torch.randn(vocab, hidden, generator=g, device=dev) / hidden**0.5
    h[:, 0], w[:, 0], w[0] = 1.0, -24.0, 0.0
    gl = torch.rand(rows, generator=g, device=dev) + 0.25
    ge = torch.randn(rows, generator=g, device=dev) * 0.1
    return labels.to(dev), h.to(dtype), w.to(dtype), gl, ge


def _half_step(x, dtype):
    """Half the distance between the two numbers of `dtype` that enclose x."""
    info = torch.finfo(dtype)
    e = torch.floor(torch.log2(x.abs().clamp_min(info.smallest_normal)))
    return torch.exp2(e) * (info.eps / 2)


def _label_exact(y, h, w, gl, ge, cap):
    """Gradients in 64 bits, tolerances under which the label's element of d
    carries no 16-bit rounding, and the gradients of a d that does.

    Off the label an element of d is off by (u + 2 dz + 2^-20) |a| p; at the
    label by (2 dz + 2^-20) |a| p + 2^-22 |b| (one float32 subtraction, and the
    part rounding took held in float32); float32 sums as in ``_exact``; the
    output by half a step at most of the number that it rounds, |x| + the rest of
    the tolerance (which may stand in the binade above x).  In dW a token with more than ``cap`` labels keeps
    its roundings."""
    keep = y >= 0
    hd = torch.where(keep[:, None], h.double(), 0.0)
    wd = w.double()
    z = hd @ wd.T
    p = torch.exp(z - torch.logsumexp(z, 1)[:, None])
    at = torch.where(keep, y, 0)
    one = torch.zeros_like(z).scatter_(1, at[:, None], 1.0)
    a, b = (gl + ge).double() * keep, gl.double() * keep
    d = a[:, None] * p - b[:, None] * one
    N, V, H = h.shape[0], w.shape[0], h.shape[1]
    dz = (H / 16 + 16) * 2.0**-22 * (hd.abs() @ wd.abs().T).amax(1)
    u = torch.finfo(h.dtype).eps / 2
    fp16 = h.dtype == FP16
    sub = 2.0**-25 if fp16 else 0.0
    dsub = sub * float(torch.maximum(a.abs(), b.abs()).max()) * 2.0**-12
    exactly = (2 * dz[:, None] + 2.0**-20) * a.abs()[:, None] * p + 2.0**-22 * b.abs()[:, None] * one
    off = exactly + u * a.abs()[:, None] * p * (1 - one) + dsub * (1 - one)
    many = torch.bincount(at[keep], minlength=V) > cap
    off_w = off + u * d.abs() * one * many[None]
    dabs = d.abs()
    top_h, top_w = hd.abs(), wd.abs()
    dh, dw = d @ wd, d.T @ hd
    tol_dh = off @ top_w + (V / 16 + 80) * 2.0**-22 * (dabs @ top_w)
    tol_dw = off_w.T @ top_h + (N / 16 + 80) * 2.0**-22 * (dabs.T @ top_h)
    tol_dh = tol_dh + _half_step(dh.abs() + tol_dh, h.dtype)
    tol_dw = tol_dw + _half_step(dw.abs() + tol_dw, h.dtype)
    scale = 1.0
    if fp16:
        scale = 2.0 ** (12 - torch.floor(torch.log2(torch.maximum(a.abs(), b.abs()).max())))
    lost = (d * scale).to(h.dtype).double() / scale * one - d * one
    return (dh, dw, tol_dh, tol_dw, (dh + lost @ wd).to(h.dtype), (dw + lost.T @ hd).to(h.dtype),
            many)


def _labels(kind, rows, vocab):
    g = torch.Generator().manual_seed(rows)
    if kind == "apart":       # hardly two in 32 tokens
        return torch.randint(1, vocab, (rows,), generator=g)
    if kind == "neighbours":  # three labels for each of 32 tokens
        return 352 + torch.arange(rows) % 32
    assert kind == "flood"    # one token with most labels among 31 with one
    y = torch.full((rows,), 352 + 5)
    y[rows - 32 :] = 352 + torch.randperm(32, generator=g)
    return y


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("kind,rows,vocab,hidden", [
    ("apart", 1, 600, 72),
    ("apart", 5, 600, 264),
    ("apart", 100, 1200, 136),
    ("apart", 300, 600, 64),       # a pair's tiles
    ("neighbours", 96, 600, 520),
    ("neighbours", 20, 600, 64),
    ("flood", 131, 600, 264),
    ("flood", 400, 600, 72),
    ("flood", 40, 600, 136),
])
def test_label_rounding_is_given_back(kind, rows, vocab, hidden, dtype) -> None:
    """What rounding takes from d at the label reaches dh of every row and dW of
    every token with up to four labels, whatever labels its neighbours have."""
    y = _labels(kind, rows, vocab)
    if rows > 10:
        y[3::11] = -100
    x = _steep(rows, vocab, hidden, dtype, y)
    dh, dw, tol_dh, tol_dw, dh_lost, dw_lost, many = _label_exact(*x, cap=4)
    if kind == "flood":
        assert 0 < int(many.sum()) <= 2
    # the tolerances tell a d with its rounding from one without
    for lost, want, tol in ((dh_lost, dh, tol_dh), (dw_lost, dw, tol_dw * (1 + many[:, None] * 1e9))):
        # (one row's coefficient may happen to be nearly a 16-bit number)
        assert int(((lost.double() - want).abs() > tol).sum()) > (hidden // 16 if rows > 1 else 0)
    got = _step(*x)
    _within("grad_hidden", got[2], dh, tol_dh)
    _within("grad_weight", got[3], dw, tol_dw)


def test_label_rounding_in_pieces_of_the_vocabulary() -> None:
    y = _labels("apart", 5000, 30011)
    x = _steep(5000, 30011, 64, BF16, y)
    dh, dw, tol_dh, tol_dw, dh_lost, dw_lost, _ = _label_exact(*x, cap=4)
    for lost, want, tol in ((dh_lost, dh, tol_dh), (dw_lost, dw, tol_dw)):
        assert int(((lost.double() - want).abs() > tol).sum()) > 1000
    got = _step(*x)
    _within("grad_hidden", got[2], dh, tol_dh)
    _within("grad_weight", got[3], dw, tol_dw)


@pytest.mark.parametrize("scale,small", [(65536.0, 2.0**-8), (1e-6, 1.0)])
def test_loss_scales_of_fp16_training(scale, small) -> None:
    """A loss scale of 65536 (on inputs small enough for the outputs' range) and
    position weights of 1e-6."""
    y, h, w, gl, ge = _inputs(100, 3000, 64, FP16)
    _check(y, h * small, w * small, gl * scale, ge * scale)


def test_coefficients_of_many_binades_in_fp16() -> None:
    """Rows whose coefficients span 2^30: one power of two serves all of them, so
    elements of d keep an absolute 2^-37 of the largest coefficient (the term
    ``dsub`` of the tolerances)."""
    y, h, w, gl, ge = _inputs(160, 3000, 64, FP16)
    s = torch.exp2(5.0 - torch.arange(160, device=h.device) % 31)
    _check(y, h, w, gl * s, ge * s)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
def test_not_finite_coefficients_stay_in_their_rows(bad, dtype) -> None:
    """An output gradient that is not finite (a loss scale too large for one row)
    makes its own row of dh not finite and leaves the other rows the bits they have
    beside a row without a gradient; dW takes the row in."""
    y, h, w, gl, ge = _inputs(150, 3000, 64, dtype, "all")
    gl, ge = gl * 1e-3, ge * 1e-3
    gl[7] = ge[7] = 0.0
    want = _step(y, h, w, gl, ge)
    for through_loss in (True, False):
        gl2, ge2 = gl.clone(), ge.clone()
        (gl2 if through_loss else ge2)[7] = bad
        got = _step(y, h, w, gl2, ge2)
        others = torch.arange(150, device=h.device) != 7
        assert torch.equal(got[2][others], want[2][others])
        assert not bool(got[2][7].isfinite().any()) and not bool(got[3].isfinite().any())


@pytest.mark.parametrize("one_,other", [((239, 29487, 16), (2, 160, 80)),
                                        ((219, 13765, 16), (321, 246, 968)),
                                        ((300, 4000, 64), (100, 3000, 64))])
def test_short_kernels_of_two_streams(one_, other) -> None:
    """Calls of more than 128 rows (CTA pairs) on one stream and of any number on
    another, again and again: their kernels follow one another on the same SMs, and the
    CTAs of a pair start and end apart."""
    x, x2 = _inputs(*one_, BF16, "all"), _inputs(*other, FP16, seed=4)
    want, want2 = _step(*x), _step(*x2)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(300):
        a, b = [], []
        for _ in range(4):
            with torch.cuda.stream(s1):
                a.append(_step(*x))
            with torch.cuda.stream(s2):
                b.append(_step(*x2))
        torch.cuda.synchronize()
        for got, ref in ((a, want), (b, want2)):
            for one in got:
                for p, q in zip(one, ref):
                    assert torch.equal(p, q)


@pytest.mark.filterwarnings("ignore:There is a performance drop")
def test_vmap_is_the_loop() -> None:
    import cid_engine

    y, h, w, gl, _ = _inputs(60, 400, 64, BF16)
    loss, lse, dh, dw = _step(y, h, w, gl, torch.zeros_like(gl))
    hr, wr = h.clone().requires_grad_(), w.clone().requires_grad_()
    l2, e2 = torch.vmap(lambda a, b: cid_engine.lm_head_cross_entropy(a, b, wr))(
        y.view(3, 20), hr.view(3, 20, 64))
    assert torch.equal(l2.detach().view(60), loss) and torch.equal(e2.detach().view(60), lse)
    dh2, _ = torch.autograd.grad(l2, (hr, wr), grad_outputs=gl.view(3, 20))
    assert torch.equal(dh2, dh)
