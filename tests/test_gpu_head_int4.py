"""The LM head with 4-bit weights: quantiser, logits and display statistics
against their formulas in 64 bits.

Tolerances: codes, scales and dequantised weights are exact.  A logit is a
float32 sum of groups: at most H / 16 + G + 16 steps (G groups) of 2^-22 of
sum |w h|, called dz; written logits add half a step of their type (and half the
smallest fp16 subnormal).  A probability exp(z - lse) moves by a relative 2 dz
plus 2^-18 for the exponentials, the sums and the merges of the parts.  The
argmax is the reference's wherever the first two logits are further apart than
2 dz.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16
SHIFTS = (0, 16, 4, 20, 8, 24, 12, 28)


@pytest.fixture(scope="module", autouse=True)
def _engine():
    import cid_engine  # noqa: F401

    assert torch.cuda.is_available()
    yield
    torch.cuda.empty_cache()


def _weight(vocab, hidden, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + vocab + 3 * hidden)
    return (torch.randn(vocab, hidden, generator=g, device="cuda") * (2.0 / hidden**0.5)).to(dtype)


def _quantized(weight, group):
    """Codes (float64) and scales (the weight's dtype) by the definition."""
    V, H = weight.shape
    w = weight.double().view(V, H // group, group)
    scales = (w.abs().amax(-1) / 7).to(weight.dtype)
    s = scales.double()[..., None]
    q = torch.where((s > 0) & s.isfinite(), torch.round(w / s), 0.0).nan_to_num(0.0).clamp(-8, 7)
    return q.view(V, H), scales


def _unpack(packed):
    V, words = packed.shape
    sh = torch.tensor(SHIFTS, device=packed.device)
    return (((packed.long()[..., None] >> sh) & 15) - 8).view(V, words * 8).double()


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("vocab,hidden,group", [
    (1, 32, 32), (3, 64, 64), (7, 128, 128), (129, 96, 32), (1001, 1600, 32), (515, 4096, 128),
    (40000, 192, 64)])
def test_quantize_is_exact(vocab, hidden, group, dtype) -> None:
    import cid_engine

    w = _weight(vocab, hidden, dtype)
    w.view(-1)[::7] *= 4  # groups of several sizes
    w[0, :group] = 0  # a group of zeros
    q, scales = _quantized(w, group)
    head = cid_engine.lm_head_quantize(w, group_size=group)
    assert head.packed.shape == (vocab, hidden // 8) and head.packed.dtype == torch.int32
    assert head.scales.dtype == dtype and torch.equal(head.scales, scales)
    assert torch.equal(_unpack(head.packed), q)
    back = cid_engine.lm_head_dequantize(*head)
    values = (q.view(vocab, -1, group) * scales.double()[..., None]).view(vocab, hidden)
    assert back.dtype == dtype and torch.equal(back, values.to(dtype))


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_quantize_rounds_ties_to_even(dtype) -> None:
    """Quotients exactly between two codes, of both signs, for many scales."""
    import cid_engine

    s = torch.tensor([1.0, 0.75, 1.171875, 2.0**-6, 1.9921875, 96.0], device="cuda")
    k = torch.arange(-7, 7, device="cuda") + 0.5
    w = torch.zeros(6, 64, device="cuda")
    w[:, 0] = 7 * s
    w[:, 1:15] = k * s[:, None]
    w[:, 15:29] = -k * s[:, None]
    wt = w.to(dtype)
    exact = (wt.float() == w).all(1)
    assert int(exact.sum()) >= 3
    head = cid_engine.lm_head_quantize(wt, group_size=64)
    q, scales = _quantized(wt, 64)
    assert torch.equal(head.scales, scales) and torch.equal(_unpack(head.packed), q)


def test_quantize_every_bf16_quotient() -> None:
    """Every bf16 value from 2^-4 to 8 against every scale mantissa: no code
    differs from the quotient in 64 bits."""
    import cid_engine

    values = torch.arange(0x3D80, 0x4100, dtype=torch.int16, device="cuda").view(BF16)  # 896 of them
    values = torch.cat([values, -values])
    tops = torch.arange(0x40E0, 0x4160, dtype=torch.int16, device="cuda").view(BF16)  # 7 to 14
    per = 31
    rows = -(-values.numel() // per)
    pad = torch.zeros(rows * per, dtype=BF16, device="cuda")
    pad[: values.numel()] = values
    w = torch.empty(tops.numel(), rows, 32, dtype=BF16, device="cuda")
    w[:, :, 0] = tops[:, None]
    w[:, :, 1:] = pad.view(1, rows, per)
    w = w.view(-1, 32)
    w[:, 1:] = torch.where(w[:, 1:].abs() > w[:, :1], w[:, :1], w[:, 1:])
    head = cid_engine.lm_head_quantize(w, group_size=32)
    q, scales = _quantized(w, 32)
    assert torch.equal(head.scales, scales) and torch.equal(_unpack(head.packed), q)


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_quantize_not_finite_and_tiny(dtype) -> None:
    import cid_engine

    w = _weight(8, 128, dtype)
    w[1, 40], w[2, 3], w[3, 100] = float("nan"), float("inf"), -float("inf")
    w[4] = 0
    w[4, 5] = torch.finfo(dtype).smallest_normal / 64  # subnormal
    w[5, :64] = torch.finfo(dtype).max
    head = cid_engine.lm_head_quantize(w, group_size=64)
    q, scales = _quantized(w, 64)
    assert torch.equal(head.scales.isnan(), scales.isnan())
    assert torch.equal(head.scales.nan_to_num(7.0), scales.nan_to_num(7.0))
    assert torch.equal(_unpack(head.packed), q)
    assert not bool(_unpack(head.packed)[1, :64].any())


def _inputs(rows, vocab, hidden, group, dtype, seed=0):
    import cid_engine

    w = _weight(vocab, hidden, dtype, seed)
    g = torch.Generator(device="cuda").manual_seed(seed + rows)
    h = torch.randn(rows, hidden, generator=g, device="cuda").to(dtype)
    ids = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    head = cid_engine.lm_head_quantize(w, group_size=group)
    values = (_unpack(head.packed).view(vocab, -1, group) * head.scales.double()[..., None])
    values = values.view(vocab, hidden)
    z = h.double() @ values.T
    dz = (hidden / 16 + hidden / group + 16) * 2.0**-22 * (h.double().abs() @ values.abs().T)
    return ids, h, head, z, dz


SIZES = [
    (1, 1, 32, 32),
    (1, 127, 64, 32),
    (3, 129, 256, 128),     # a weight row past a tile
    (16, 1000, 288, 32),    # a K tail of a chunk
    (17, 1000, 320, 64),    # two passes of 16 or one of 32
    (33, 777, 640, 128),    # 64-row pass, mostly empty
    (40, 513, 384, 64),
    (64, 5003, 1024, 128),
    (130, 2049, 512, 128),  # three passes of 64 rows
    (50, 1500, 1600, 32),   # four passes of 16
    (5, 20000, 2048, 64),   # more tiles than SMs
    (70, 40000, 512, 128),  # several tiles and passes a CTA
    (20, 40000, 4096, 128), # hidden rows too many for shared memory
    (64, 80000, 1536, 128), # the same, several tiles of 256 weight rows a CTA
    (16, 3000, 8192, 32),
    (9, 9999, 4096, 128),   # 16 rows a pass, 15 weight rows in the last tile
    (8, 30011, 1152, 64),   # the small-row kernel, nine blocks of columns
    (2, 70001, 96, 32),     # one block of columns; groups of 32 take the other kernel
]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("rows,vocab,hidden,group", SIZES)
def test_logits(rows, vocab, hidden, group, dtype) -> None:
    import cid_engine

    cid_engine.device_status(0, reset=True)
    _, h, head, z, dz = _inputs(rows, vocab, hidden, group, dtype)
    got = cid_engine.lm_head_quantized_logits(h, *head)
    assert got.shape == (rows, vocab) and got.dtype == dtype
    u = torch.finfo(dtype).eps / 2
    off = (got.double() - z).abs()
    tol = dz * (1 + u) + u * z.abs() + (2.0**-25 if dtype == FP16 else 0.0)
    assert bool((off <= tol).all()), f"worst {float((off / tol).max()):.3g} of the tolerance"
    assert cid_engine.device_status(0) == 0


def _check_stats(ids, h, head, z, dz):
    import cid_engine

    cid_engine.device_status(0, reset=True)
    conf, pred, cur = cid_engine.lm_head_quantized_display_statistics(ids, h, *head, round_bf16=False)
    p = torch.softmax(z, 1)
    rel = 2 * dz.amax(1) + 2.0**-18
    e_conf, e_cur = p.amax(1), p.gather(1, ids[:, None])[:, 0]
    assert bool(((conf.double() - e_conf).abs() <= rel * 1.01 * e_conf).all())
    assert bool(((cur.double() - e_cur).abs() <= rel * 1.01 * e_cur + 1e-38).all())
    held = z.gather(1, pred[:, None])[:, 0]
    top = z.amax(1)
    assert bool((top - held <= 2 * dz.amax(1)).all())
    if z.shape[1] > 1:
        two = z.topk(2, 1).values
        clear = two[:, 0] - two[:, 1] > 2 * dz.amax(1)
        assert bool(clear.any()) and torch.equal(pred[clear], z.argmax(1)[clear])
    assert cid_engine.device_status(0) == 0
    return conf, pred, cur


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("rows,vocab,hidden,group", SIZES)
def test_statistics(rows, vocab, hidden, group, dtype) -> None:
    _check_stats(*_inputs(rows, vocab, hidden, group, dtype))


def test_rounded_statistics_are_those_of_the_written_logits() -> None:
    """With round_bf16 the statistics are those of the bf16 logits the product
    writes: the two come from the same sums."""
    import cid_engine

    ids, h, head, _, _ = _inputs(48, 9000, 1024, 128, BF16)
    logits = cid_engine.lm_head_quantized_logits(h, *head)
    want = cid_engine.display_token_statistics(ids[None], logits[None])
    got = cid_engine.lm_head_quantized_display_statistics(ids, h, *head)
    assert torch.equal(got[1], want[1][0])
    # the same logits, summed in another order: relative 2^-18
    torch.testing.assert_close(got[0], want[0][0], rtol=2.0**-18, atol=0)
    torch.testing.assert_close(got[2], want[2][0], rtol=2.0**-18, atol=1e-38)


def test_equal_columns_take_the_lower_one() -> None:
    import cid_engine

    ids, h, head, _, _ = _inputs(40, 3000, 256, 64, BF16)
    packed, scales = head.packed.clone(), head.scales.clone()
    for a, b in ((17, 2900), (17, 1500), (599, 600), (127, 128)):
        packed[b], scales[b] = packed[a], scales[a]
    logits = cid_engine.lm_head_quantized_logits(h, packed, scales)
    assert torch.equal(logits[:, 17], logits[:, 2900])
    h2 = h.clone()
    # rows that point at column 17, 599 or 127
    w = cid_engine.lm_head_dequantize(packed, scales)
    for r in range(40):
        h2[r] = (w[(17, 599, 127)[r % 3]].float() * 8).to(BF16)
    _, pred, _ = cid_engine.lm_head_quantized_display_statistics(ids, h2, packed, scales)
    assert pred.tolist() == [(17, 599, 127)[r % 3] for r in range(40)]


def test_not_finite_values() -> None:
    """A NaN hidden row has NaN statistics and its neighbours none; a NaN scale
    makes its column NaN for every row, and the argmax the first of them."""
    import cid_engine

    ids, h, head, _, _ = _inputs(20, 2000, 256, 128, BF16)
    want = cid_engine.lm_head_quantized_display_statistics(ids, h, *head)
    h2 = h.clone()
    h2[7, 100] = float("nan")
    got = cid_engine.lm_head_quantized_display_statistics(ids, h2, *head)
    assert bool(got[0][7].isnan()) and int(got[1][7]) == 0
    keep = torch.arange(20, device="cuda") != 7
    for a, b in zip(got, want):
        assert torch.equal(a[keep], b[keep])
    scales = head.scales.clone()
    scales[1333, 1], scales[1700, 0] = float("nan"), float("nan")
    logits = cid_engine.lm_head_quantized_logits(h, head.packed, scales)
    assert torch.equal(logits.isnan().nonzero()[:, 1].unique().cpu(), torch.tensor([1333, 1700]))
    conf, pred, _ = cid_engine.lm_head_quantized_display_statistics(ids, h, head.packed, scales)
    assert bool(conf.isnan().all()) and bool((pred == 1333).all())


def test_out_of_range_ids_set_the_status() -> None:
    import cid_engine

    ids, h, head, _, _ = _inputs(20, 500, 128, 64, BF16)
    ids[3], ids[9] = 500, -1
    cid_engine.device_status(0, reset=True)
    conf, _, cur = cid_engine.lm_head_quantized_display_statistics(ids, h, *head)
    assert cur.isnan().nonzero().flatten().tolist() == [3, 9] and not bool(conf.isnan().any())
    assert cid_engine.device_status(0, reset=True) == cid_engine.STATUS_TOKEN_ID_OUT_OF_RANGE


def test_shapes_views_and_repeats() -> None:
    import cid_engine

    ids, h, head, _, _ = _inputs(24, 900, 256, 64, BF16)
    logits = cid_engine.lm_head_quantized_logits(h, *head)
    stats = cid_engine.lm_head_quantized_display_statistics(ids, h, *head)
    for _ in range(2):
        assert torch.equal(cid_engine.lm_head_quantized_logits(h, *head), logits)
    wide = torch.zeros(24, 300, dtype=BF16, device="cuda")
    wide[:, 3:259] = h
    pt = head.packed.T.contiguous().T
    st = torch.stack([head.scales, head.scales], -1)[..., 0]
    off = torch.empty(900 * 32 + 1, dtype=torch.int32, device="cuda")[1:].view(900, 32)
    off.copy_(head.packed)
    assert torch.equal(cid_engine.lm_head_quantized_logits(wide[:, 3:259], pt, st), logits)
    assert torch.equal(cid_engine.lm_head_quantized_logits(h, off, head.scales), logits)
    b = cid_engine.lm_head_quantized_logits(h.view(2, 3, 4, 256), *head)
    assert b.shape == (2, 3, 4, 900) and torch.equal(b.view(24, 900), logits)
    assert torch.equal(cid_engine.lm_head_quantized_logits(h[5], *head), logits[5])
    s2 = cid_engine.lm_head_quantized_display_statistics(ids.view(4, 6), h.view(4, 6, 256), *head)
    for a, c in zip(s2, stats):
        assert a.shape == (4, 6) and torch.equal(a.view(-1), c)
    assert cid_engine.lm_head_quantized_logits(h[:0], *head).shape == (0, 900)
    e = cid_engine.lm_head_quantized_display_statistics(ids[:0], h[:0], *head)
    assert [t.shape for t in e] == [(0,)] * 3
    w = _weight(30, 128, BF16)
    odd = torch.empty(30 * 128 + 1, dtype=BF16, device="cuda")[1:].view(30, 128)
    odd.copy_(w)
    for a, c in zip(cid_engine.lm_head_quantize(odd), cid_engine.lm_head_quantize(w)):
        assert torch.equal(a, c)


def test_two_streams_and_graph_replay() -> None:
    import cid_engine

    a, b = _inputs(30, 4000, 512, 128, BF16), _inputs(9, 7000, 256, 32, FP16, seed=2)

    def both(x):
        return (cid_engine.lm_head_quantized_logits(x[1], *x[2]),
                *cid_engine.lm_head_quantized_display_statistics(x[0], x[1], *x[2]))

    want = both(a), both(b)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(4):
        with torch.cuda.stream(s1):
            ga = both(a)
        with torch.cuda.stream(s2):
            gb = both(b)
        torch.cuda.synchronize()
        for got, ref in zip((ga, gb), want):
            for p, q in zip(got, ref):
                assert torch.equal(p, q)
    h = a[1].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both((a[0], h, a[2]))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both((a[0], h, a[2]))
    h.copy_(a[1].flip(0))
    graph.replay()
    for p, q in zip(out, both((a[0], a[1].flip(0), a[2]))):
        assert torch.equal(p, q)


def test_train_quantize_decode() -> None:
    """The operators as one run: a training step of the head on corrupted
    display rows, the trained weight laid out in 4 bits, and the decode step and
    loop on it, equal to the steps put together by hand."""
    import cid_engine

    dev = torch.device("cuda", 0)
    g = torch.Generator(device=dev).manual_seed(8)
    B, L, V, H = 2, 40, 1536, 256
    ids = torch.randint(2, V, (B, L), generator=g, device=dev)
    hidden = torch.randn(B, L, H, generator=g, device=dev).to(BF16)
    weight = _weight(V, H, BF16).requires_grad_()
    corrupted, labels, _, _ = cid_engine.display_corrupt_from_random(
        ids, torch.full((B,), 0.5, device=dev), torch.ones(B, L, dtype=torch.bool, device=dev),
        torch.rand(B, L, generator=g, device=dev), None, None, mask_token_id=0, eos_token_id=1,
        vocab_size=V, replacement_fraction=0.0)
    loss, _ = cid_engine.lm_head_cross_entropy(labels, hidden, weight)
    loss.sum().backward()
    with torch.no_grad():
        trained = (weight - 0.5 * weight.grad).detach()
    head = cid_engine.lm_head_quantize(trained, group_size=64)
    kw = dict(mask_token_id=0, eos_token_id=1, reveal_fraction=0.3, revision_fraction=0.1,
              revision_margin=0.05)
    out = cid_engine.refine_step_from_hidden(corrupted, hidden, head, **kw)
    stats = cid_engine.lm_head_quantized_display_statistics(corrupted, hidden, *head)
    refined = cid_engine.refine_display_from_statistics(corrupted, *stats, **kw)
    assert torch.equal(out.token_ids, refined) and torch.equal(out.predicted, stats[1])
    assert int((refined != 0).sum()) > int((corrupted != 0).sum())
    for graphs in (False, True):
        loop = cid_engine.DisplayRefineLoop(corrupted, [hidden], lm_head_weight=head,
                                            use_graphs=graphs, **kw)
        loop.run(3)
        by_hand = corrupted
        for _ in range(3):
            by_hand = cid_engine.refine_step_from_hidden(by_hand, hidden, head, **kw).token_ids
        torch.cuda.synchronize()
        assert torch.equal(loop.ids, by_hand)


@pytest.mark.parametrize("rows", [3, 40])
def test_fp16_hidden_rows_rounded_to_bf16(rows) -> None:
    """round_bf16 rounds the float32 logits to bfloat16 whatever the hidden type."""
    import cid_engine

    ids, h, head, z, dz = _inputs(rows, 3000, 256, 64, FP16)
    conf, pred, _ = cid_engine.lm_head_quantized_display_statistics(ids, h, *head)
    zb = z.to(BF16).double()
    p = torch.softmax(zb, 1).amax(1)
    # a logit near a rounding border may fall on the other side: one step of it
    step = zb.abs().amax(1) * 2.0**-7
    assert bool(((conf.double() - p).abs() <= (2 * dz.amax(1) + 2 * step) * p).all())
    held = zb.gather(1, pred[:, None])[:, 0]
    assert bool((zb.amax(1) - held <= step).all())


@pytest.mark.parametrize("rows,dtype", [(4, BF16), (30, BF16), (4, FP16), (30, FP16)])
def test_hidden_rows_of_every_size(rows, dtype) -> None:
    """Rows from the type's subnormals to its largest values, and rows whose
    elements span its range: the power of two that a row is scaled by is undone."""
    import cid_engine

    _, h, head, _, _ = _inputs(rows, 600, 256, 128, dtype)
    tiny, big = torch.finfo(dtype).smallest_normal, torch.finfo(dtype).max
    scale = torch.logspace(-1, 1, rows, device="cuda", dtype=torch.float64)
    h = h.double()
    h[0] *= tiny / 8
    h[1] *= big / 1e6
    h[2, ::3] *= 1e-4
    h[3] = 0
    h = (h * scale[:, None]).to(dtype)
    got = cid_engine.lm_head_quantized_logits(h, *head).double()
    V = head.packed.shape[0]
    values = (_unpack(head.packed).view(V, 2, 128) * head.scales.double()[..., None]).view(V, 256)
    z = h.double() @ values.T
    dz = (256 / 16 + 2 + 16) * 2.0**-22 * (h.double().abs() @ values.abs().T)
    # elements below 2^-24 of their row's largest lose up to 2^-35 of it
    dz += 2.0**-35 * h.double().abs().amax(1)[:, None] * values.abs().sum(1)[None]
    u = torch.finfo(dtype).eps / 2
    ok = z.abs() < big * 0.99
    tol = dz * (1 + u) + u * z.abs() + torch.finfo(dtype).smallest_normal * u * 2 + 2.0**-149
    assert bool(((got - z).abs() <= tol)[ok].all())
    assert not bool(got[3].any())


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("rows,vocab,hidden,group", [
    # hidden rows in shared memory, 16 a pass, two groups a chunk
    (12, 1000, 320, 64),
    (16, 40000, 2112, 64),
    # hidden rows streamed beside the codes, one and two tiles of 256 weight rows a CTA
    (24, 40000, 4096, 64),
    (12, 40000, 5184, 64),   # a K tail of a chunk
    (12, 40000, 8192, 128),
    (16, 40000, 8224, 32),
    (33, 3000, 32768, 128),  # the widest hidden rows
    (32, 3000, 32768, 64),
    (16, 3000, 32768, 32),
    (5, 3000, 32768, 128),   # 8 rows that do not fit the small-row kernel
    (8, 1001, 16384, 64),
    # the small-row kernel with half a block of columns at the end
    (4, 3000, 64, 64),
    (7, 1000, 192, 64),
    (8, 20000, 1088, 64),
    (1, 129, 64, 64),
])
def test_every_form_of_the_products(rows, vocab, hidden, group, dtype) -> None:
    """Sizes that reach the forms of the two product kernels beside those above,
    for the logits and for the statistics."""
    import cid_engine

    cid_engine.device_status(0, reset=True)
    ids, h, head, z, dz = _inputs(rows, vocab, hidden, group, dtype)
    got = cid_engine.lm_head_quantized_logits(h, *head)
    u = torch.finfo(dtype).eps / 2
    off = (got.double() - z).abs()
    tol = dz * (1 + u) + u * z.abs() + (2.0**-25 if dtype == FP16 else 0.0)
    assert bool((off <= tol).all()), f"worst {float((off / tol).max()):.3g} of the tolerance"
    _check_stats(ids, h, head, z, dz)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("rows,group", [(4, 128), (4, 64), (4, 32), (20, 128), (20, 64), (50, 128),
                                        (50, 32)])
def test_infinite_weights_make_their_columns_nan(rows, group, dtype) -> None:
    """An infinite weight leaves its group an infinite scale and codes 0: 0 x inf,
    a NaN logit in every row, and NaN statistics with the first such column."""
    import cid_engine

    w = _weight(2000, 512, dtype)
    w[1333, 5], w[1700, 400] = float("inf"), -float("inf")
    head = cid_engine.lm_head_quantize(w, group_size=group)
    g = torch.Generator(device="cuda").manual_seed(rows)
    # values off zero on one side, so that sums of h are large beside their roundings
    h = (torch.randn(rows, 512, generator=g, device="cuda") + 0.3).to(dtype)
    logits = cid_engine.lm_head_quantized_logits(h, *head)
    assert int(logits.isnan().sum()) == 2 * rows and not bool(logits.isinf().any())
    assert bool(logits[:, [1333, 1700]].isnan().all())
    conf, pred, cur = cid_engine.lm_head_quantized_display_statistics(
        torch.zeros(rows, dtype=torch.long, device="cuda"), h, *head)
    assert bool(conf.isnan().all()) and bool((pred == 1333).all()) and bool(cur.isnan().all())


@pytest.mark.parametrize("rows,vocab,hidden,group,dtype", [
    (15, 37889, 2048, 32, FP16),
    (1, 34741, 4096, 32, FP16),
    (93, 18944, 3584, 32, BF16),
    (135, 37888, 3456, 32, BF16),
    (65, 2653, 2048, 64, BF16),
    (64, 18945, 1024, 128, BF16),
])
def test_stages_are_refilled_after_they_are_read(rows, vocab, hidden, group, dtype) -> None:
    """Where the read-back of many scales holds the loads of an SM up, a stage of
    codes that is handed back before its loads have come in holds other columns'
    codes for some weight rows.  Several operands at other addresses, each called
    again and again: every call gives the oracle's logits and the first call's bits."""
    import cid_engine

    keep = []
    for seed in range(4):
        _, h, head, z, dz = _inputs(rows, vocab, hidden, group, dtype, seed)
        keep.append((h, head))  # the next operands stand elsewhere
        u = torch.finfo(dtype).eps / 2
        tol = dz * (1 + u) + u * z.abs() + (2.0**-25 if dtype == FP16 else 0.0)
        first = cid_engine.lm_head_quantized_logits(h, *head)
        assert bool(((first.double() - z).abs() <= tol).all())
        for _ in range(8):
            assert torch.equal(cid_engine.lm_head_quantized_logits(h, *head), first)


@pytest.mark.parametrize("rows,vocab,hidden,group", [
    (64, 40001, 1024, 128), (40, 40001, 1024, 128), (32, 30011, 2048, 64), (12, 20011, 4352, 64),
    (16, 20011, 4224, 32)])
def test_late_loads_of_codes(rows, vocab, hidden, group) -> None:
    """Sizes at which shared memory has room for nine stages of codes, while copies on
    another stream delay some of their loads: the first call's bits every time."""
    import cid_engine

    _, h, head, z, dz = _inputs(rows, vocab, hidden, group, BF16)
    first = cid_engine.lm_head_quantized_logits(h, *head)
    u = torch.finfo(BF16).eps / 2
    assert bool(((first.double() - z).abs() <= dz * (1 + u) + u * z.abs()).all())
    big = torch.zeros(1 << 28, dtype=torch.uint8, device="cuda")
    other = torch.empty_like(big)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(40):
            other.copy_(big)
    got = [cid_engine.lm_head_quantized_logits(h, *head) for _ in range(24)]
    torch.cuda.synchronize()
    assert all(torch.equal(g, first) for g in got)
