"""The LM head's training and 4-bit operators on the host: schemas, refusals,
shapes on the meta device, autograd, and the C ABI's checks (no GPU)."""

from __future__ import annotations

import ctypes
import importlib.util
from pathlib import Path

import pytest
import torch

import cid_engine

ROOT = Path(__file__).resolve().parent.parent
LIB = ROOT / "cid-engine_b200" / "cid_engine" / "libcid_engine_b200.so"
OK, INVALID, DTYPE, MISALIGNED, SCRATCH = 0, 1, 2, 4, 6
F32, F16, BF16 = 0, 2, 3


@pytest.fixture(scope="module")
def lib() -> ctypes.CDLL:
    lib = ctypes.CDLL(str(LIB))
    lib.cid_lm_head_cross_entropy_workspace_bytes.restype = ctypes.c_size_t
    lib.cid_lm_head_quantized_workspace_bytes.restype = ctypes.c_size_t
    return lib


def _loss_inputs(device="cpu", dtype=torch.bfloat16, grad=False):
    y = torch.zeros(3, 5, dtype=torch.long, device=device)
    h = torch.zeros(3, 5, 64, dtype=dtype, device=device, requires_grad=grad)
    w = torch.zeros(100, 64, dtype=dtype, device=device, requires_grad=grad)
    return y, h, w


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_loss_shapes_and_gradients_on_meta(dtype) -> None:
    y, h, w = _loss_inputs("meta", dtype, grad=True)
    loss, lse = cid_engine.lm_head_cross_entropy(y, h, w)
    for t in (loss, lse):
        assert t.shape == (3, 5) and t.dtype == torch.float32 and t.requires_grad
    gh, gw = torch.autograd.grad(loss.mean() + (lse**2).mean(), (h, w))
    assert gh.shape == h.shape and gw.shape == w.shape and gh.dtype == gw.dtype == dtype
    for ignore in (-100, 7):  # the default and another value take the same path
        loss, _ = cid_engine.lm_head_cross_entropy(y, h.detach(), w, ignore_index=ignore)
        (gw,) = torch.autograd.grad(loss.sum(), w)
        assert gw.shape == w.shape
    loss, _ = cid_engine.lm_head_cross_entropy(y, h.detach(), w.detach())
    assert not loss.requires_grad


def test_loss_has_no_second_gradient() -> None:
    y, h, w = _loss_inputs("meta", grad=True)
    loss, _ = cid_engine.lm_head_cross_entropy(y, h, w)
    gh, _ = torch.autograd.grad(loss.sum(), (h, w), create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(gh.sum(), h)


def test_loss_refusals() -> None:
    y, h, w = _loss_inputs()
    f = cid_engine.lm_head_cross_entropy
    with pytest.raises(RuntimeError, match="CUDA devices only"):
        f(y, h, w)
    with pytest.raises(RuntimeError, match="labels must use torch.int64"):
        f(y.int(), h, w)
    with pytest.raises(RuntimeError, match=r"\[\*labels.shape, hidden_dim\]"):
        f(y[:2], h, w)
    with pytest.raises(RuntimeError, match=r"\[vocab, hidden_dim\]"):
        f(y, h, w[:, :56])
    with pytest.raises(RuntimeError, match="both"):
        f(y, h, w.half())
    with pytest.raises(RuntimeError, match="both"):
        f(y, h.float(), w.float())
    with pytest.raises(RuntimeError, match="non-empty"):
        f(y, h, w[:0])
    with pytest.raises(RuntimeError, match="multiple of 8"):
        f(y, h[..., :60], w[:, :60])
    with pytest.raises(RuntimeError, match="same device"):
        f(y.to("meta"), h, w)
    b = torch.ops.cid_engine.lm_head_cross_entropy_backward
    g = torch.zeros(3, 5)
    with pytest.raises(RuntimeError, match="log_sum_exp"):
        b(g, None, y, h, w, torch.zeros(3), -100, True, True)
    with pytest.raises(RuntimeError, match="output gradients"):
        b(g.double(), None, y, h, w, g, -100, True, True)
    with pytest.raises(RuntimeError, match="CUDA devices only"):
        b(g, None, y, h, w, g, -100, True, True)


def test_loss_c_abi_checks(lib: ctypes.CDLL) -> None:
    i64, p, null, size = ctypes.c_int64, ctypes.c_void_p, ctypes.c_void_p(0), ctypes.c_size_t
    ws = lib.cid_lm_head_cross_entropy_workspace_bytes

    def need(rows, dim, vocab, backward):
        return ws(i64(rows), i64(dim), i64(vocab), ctypes.c_int(backward))

    assert 0 < need(4, 64, 300, 0) < need(4, 64, 300, 1)
    for bad in ((0, 64, 300), (-1, 64, 300), (4, 60, 300), (4, 0, 300), (4, 64, 0), (4, 64, 2**31 - 1),
                (2**31, 64, 300), (2**30, 2**30, 300)):
        assert need(*bad, 0) == 0

    def loss(dtype=BF16, rows=4, dim=64, vocab=300, h=0x1000, w=0x2000, y=0x3000, out=0x4000,
             bytes_=1 << 40):
        return lib.cid_lm_head_cross_entropy(
            dtype, p(h), i64(rows), i64(dim), p(w), i64(vocab), p(y), i64(-100), p(out),
            p(0x5000), p(0x6000), size(bytes_), null, null)

    assert loss(dtype=F32) == DTYPE
    assert loss(dim=12) == INVALID and loss(rows=-1) == INVALID and loss(vocab=0) == INVALID
    assert loss(h=0x1008) == MISALIGNED and loss(y=0x3004) == MISALIGNED
    assert loss(out=0x4002) == MISALIGNED
    assert loss(rows=0) == OK
    assert loss(h=0) == INVALID and loss(y=0) == INVALID and loss(out=0) == INVALID
    assert loss(bytes_=need(4, 64, 300, 0) - 1) == SCRATCH

    def back(dtype=BF16, rows=4, dim=64, lse=0x4000, gl=0x4100, gh=0x5000, gw=0x6000,
             bytes_=1 << 40):
        return lib.cid_lm_head_cross_entropy_backward(
            dtype, p(0x1000), i64(rows), i64(dim), p(0x2000), i64(300), p(0x3000), i64(-100),
            p(lse), p(gl), null, p(gh), p(gw), p(0x7000), size(bytes_), null, null)

    assert back(dtype=F32) == DTYPE and back(dim=4) == INVALID
    assert back(gh=0x5008) == MISALIGNED and back(gl=0x4102) == MISALIGNED
    assert back(gh=0, gw=0) == OK  # nothing wanted
    assert back(rows=0, gw=0) == OK
    assert back(lse=0) == INVALID
    assert back(bytes_=need(4, 64, 300, 1) - 1) == SCRATCH


def _packed(device="cpu", dtype=torch.bfloat16, vocab=100, dim=128, group=64):
    return (torch.zeros(vocab, dim // 8, dtype=torch.int32, device=device),
            torch.zeros(vocab, dim // group, dtype=dtype, device=device))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_int4_shapes_on_meta(dtype, group) -> None:
    w = torch.zeros(100, 256, dtype=dtype, device="meta")
    head = cid_engine.lm_head_quantize(w, group_size=group)
    assert isinstance(head, cid_engine.QuantizedLMHead)
    assert head.packed.shape == (100, 32) and head.packed.dtype == torch.int32
    assert head.scales.shape == (100, 256 // group) and head.scales.dtype == dtype
    assert cid_engine.lm_head_dequantize(*head).shape == (100, 256)
    h = torch.zeros(3, 5, 256, dtype=dtype, device="meta")
    z = cid_engine.lm_head_quantized_logits(h, *head)
    assert z.shape == (3, 5, 100) and z.dtype == dtype
    ids = torch.zeros(3, 5, dtype=torch.long, device="meta")
    c, p, u = cid_engine.lm_head_quantized_display_statistics(ids, h, *head)
    assert c.shape == p.shape == u.shape == (3, 5)
    assert c.dtype == u.dtype == torch.float32 and p.dtype == torch.int64
    assert cid_engine.lm_head_quantize(w).scales.shape == (100, 2)


def test_int4_refusals() -> None:
    w = torch.zeros(100, 128, dtype=torch.bfloat16)
    q = cid_engine.lm_head_quantize
    with pytest.raises(RuntimeError, match="CUDA devices only"):
        q(w)
    with pytest.raises(RuntimeError, match="bfloat16 or torch.float16"):
        q(w.float())
    with pytest.raises(RuntimeError, match="32, 64 or 128"):
        q(w, group_size=16)
    with pytest.raises(RuntimeError, match="multiple of group_size"):
        q(w[:, :96], group_size=64)
    with pytest.raises(RuntimeError, match="non-empty"):
        q(w[:0])
    with pytest.raises(RuntimeError, match=r"\[vocab, hidden_dim\]"):
        q(w[0])
    packed, scales = _packed()
    for f in (lambda p, s: cid_engine.lm_head_dequantize(p, s),
              lambda p, s: cid_engine.lm_head_quantized_logits(
                  torch.zeros(2, 128, dtype=torch.bfloat16), p, s)):
        with pytest.raises(RuntimeError, match="CUDA devices only"):
            f(packed, scales)
        with pytest.raises(RuntimeError, match="packed must be an int32"):
            f(packed.long(), scales)
        with pytest.raises(RuntimeError, match="scales must be"):
            f(packed, scales.float())
        with pytest.raises(RuntimeError, match="scales must be"):
            f(packed, scales[:50])
        with pytest.raises(RuntimeError, match="groups of 32, 64 or 128"):
            f(packed, torch.zeros(100, 8, dtype=torch.bfloat16))
        with pytest.raises(RuntimeError, match="groups of 32, 64 or 128"):
            f(packed, scales[:, :0])
        with pytest.raises(RuntimeError, match="non-empty"):
            f(packed[:0], scales[:0])
    h = torch.zeros(2, 128, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="share a dtype"):
        cid_engine.lm_head_quantized_logits(h.half(), packed, scales)
    with pytest.raises(RuntimeError, match=r"\[\*, hidden_dim\]"):
        cid_engine.lm_head_quantized_logits(h[:, :64], packed, scales)
    s = cid_engine.lm_head_quantized_display_statistics
    ids = torch.zeros(2, dtype=torch.long)
    with pytest.raises(RuntimeError, match="CUDA devices only"):
        s(ids, h, packed, scales)
    with pytest.raises(RuntimeError, match="torch.int64"):
        s(ids.int(), h, packed, scales)
    with pytest.raises(RuntimeError, match=r"\[\*token_ids.shape, hidden_dim\]"):
        s(ids[:1], h, packed, scales)


def test_int4_c_abi_checks(lib: ctypes.CDLL) -> None:
    i64, p, null, size = ctypes.c_int64, ctypes.c_void_p, ctypes.c_void_p(0), ctypes.c_size_t

    def quantize(dtype=BF16, w=0x1000, vocab=100, dim=128, group=64, out=0x2000, sc=0x3000):
        return lib.cid_lm_head_quantize(dtype, p(w), i64(vocab), i64(dim), ctypes.c_int(group),
                                        p(out), p(sc), null)

    def dequantize(dtype=BF16, w=0x1000, vocab=100, dim=128, group=64, out=0x2000, sc=0x3000):
        return lib.cid_lm_head_dequantize(dtype, p(out), p(sc), i64(vocab), i64(dim),
                                          ctypes.c_int(group), p(w), null)

    for f in (quantize, dequantize):
        assert f(dtype=F32) == DTYPE
        for bad in (dict(vocab=0), dict(vocab=2**31), dict(dim=0), dict(dim=96), dict(group=16),
                    dict(group=0), dict(dim=-64), dict(vocab=2**30, dim=2**30)):
            assert f(**bad) == INVALID, bad
        assert f(w=0x1008) == MISALIGNED and f(out=0x2004) == MISALIGNED and f(sc=0x3001) == MISALIGNED
        assert f(w=0) == INVALID and f(out=0) == INVALID and f(sc=0) == INVALID

    def need(rows, dim, vocab, group, statistics):
        return lib.cid_lm_head_quantized_workspace_bytes(
            i64(rows), i64(dim), i64(vocab), ctypes.c_int(group), ctypes.c_int(statistics))

    assert 0 < need(2, 128, 300, 64, 0)
    assert need(2, 128, 300, 64, 1) == need(2, 128, 300, 64, 0) + 3 * 2 * 16
    for bad in ((0, 128, 300, 64), (-1, 128, 300, 64), (2, 0, 300, 64), (2, 128, 0, 64),
                (2, 128, 2**31, 64), (2, 128, 300, 48), (2, 32768 + 128, 300, 64)):
        assert need(*bad, 1) == 0

    def logits(dtype=BF16, rows=2, h=0x1000, dim=128, group=64, vocab=100, out=0x5000, ws=0x6000,
               bytes_=1 << 40):
        return lib.cid_lm_head_quantized_logits(dtype, p(h), i64(rows), i64(dim), p(0x2000),
                                                p(0x3000), ctypes.c_int(group), i64(vocab), p(out),
                                                p(ws), size(bytes_), null, null)

    assert logits(dtype=F32) == DTYPE and logits(rows=-1) == INVALID and logits(dim=100) == INVALID
    assert logits(rows=2**31) == INVALID and logits(h=0x1002) == MISALIGNED
    assert logits(dim=32768 + 128) == INVALID and logits(ws=0x6008) == MISALIGNED
    assert logits(out=0x5001) == MISALIGNED and logits(rows=0) == OK
    assert logits(h=0) == INVALID and logits(out=0) == INVALID and logits(ws=0) == INVALID
    assert logits(bytes_=need(2, 128, 100, 64, 0) - 1) == SCRATCH

    def stats(ids=0x4000, ws=0x6000, bytes_=1 << 40, rows=2):
        return lib.cid_lm_head_quantized_display_statistics(
            BF16, p(0x1000), i64(rows), i64(128), p(0x2000), p(0x3000), ctypes.c_int(64),
            i64(300), p(ids), ctypes.c_int(1), p(0x5000), p(0x5100), p(0x5200), p(ws),
            size(bytes_), null, null)

    assert stats(ids=0x4004) == MISALIGNED and stats(ws=0x6008) == MISALIGNED
    assert stats(ids=0) == INVALID and stats(ws=0) == INVALID and stats(rows=0) == OK
    assert stats(bytes_=need(2, 128, 300, 64, 1) - 1) == SCRATCH


@pytest.mark.parametrize("which", ["hidden", "weight"])
@pytest.mark.parametrize("recorded", [False, True])
@pytest.mark.parametrize("grad_mode", [False, True])
def test_loss_refuses_tangents(which, recorded, grad_mode) -> None:
    """A dual tensor is refused whether or not a graph is being recorded: outputs
    without a tangent would stand for a derivative of zero."""
    y, h, w = _loss_inputs("meta", grad=recorded)
    with torch.autograd.forward_ad.dual_level(), torch.set_grad_enabled(grad_mode):
        make = torch.autograd.forward_ad.make_dual
        if which == "hidden":
            h = make(h, torch.ones_like(h))
        else:
            w = make(w, torch.ones_like(w))
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            cid_engine.lm_head_cross_entropy(y, h, w)


def test_loss_refuses_forward_transforms() -> None:
    y, h, w = _loss_inputs("meta")
    with pytest.raises(RuntimeError, match="no forward-mode derivative"):
        torch.func.jvp(lambda a: cid_engine.lm_head_cross_entropy(y, a, w)[0], (h,),
                       (torch.ones_like(h),))
    with pytest.raises(RuntimeError, match="no forward-mode derivative"):
        torch.func.jacfwd(lambda a: cid_engine.lm_head_cross_entropy(y[0, :1], a, w)[0])(h[0, :1])
    with pytest.raises(RuntimeError, match="functorch"):
        torch.func.grad(lambda a: cid_engine.lm_head_cross_entropy(y, a, w)[0].sum())(h)


@pytest.mark.parametrize("place", [0, 1, 3, 4, 5])
def test_loss_backward_refuses_tangents(place) -> None:
    y, h, w = _loss_inputs("meta")
    args = [torch.zeros(3, 5, device="meta"), torch.zeros(3, 5, device="meta"), y, h, w,
            torch.zeros(3, 5, device="meta")]
    b = torch.ops.cid_engine.lm_head_cross_entropy_backward
    assert b(*args, -100, True, True)[0].shape == h.shape
    with torch.autograd.forward_ad.dual_level():
        args[place] = torch.autograd.forward_ad.make_dual(args[place], torch.ones_like(args[place]))
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            b(*args, -100, True, True)


def test_loss_backward_refuses_a_dual_output_gradient() -> None:
    y, h, w = _loss_inputs("meta", grad=True)
    loss, _ = cid_engine.lm_head_cross_entropy(y, h, w)
    with torch.autograd.forward_ad.dual_level():
        g = torch.autograd.forward_ad.make_dual(torch.ones(3, 5, device="meta"),
                                                torch.ones(3, 5, device="meta"))
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            torch.autograd.grad(loss, h, g)


@pytest.mark.filterwarnings("ignore:There is a performance drop")
def test_loss_under_vmap_keeps_shapes() -> None:
    """vmap runs the operator once for each item; a graph is recorded through it."""
    y, h, w = _loss_inputs("meta")
    h.requires_grad_()
    loss, lse = torch.vmap(lambda a, b: cid_engine.lm_head_cross_entropy(a, b, w))(y, h)
    assert loss.shape == lse.shape == (3, 5) and loss.requires_grad
    (gh,) = torch.autograd.grad(loss.sum(), h)
    assert gh.shape == h.shape


def test_loss_workspace_follows_the_call(lib: ctypes.CDLL) -> None:
    """The backward's workspace holds a piece of the logits' gradient and the parts
    of dh that the extents can make, not the most that any can."""
    i64 = ctypes.c_int64

    def need(rows, dim, vocab):
        return lib.cid_lm_head_cross_entropy_workspace_bytes(i64(rows), i64(dim), i64(vocab),
                                                             ctypes.c_int(1))

    assert need(64, 64, 4096) < 4 << 20
    assert need(1, 8, 7) < 1 << 20
    assert need(129, 64, 4096) < 8 << 20
    # parts of dh: 592 tiles of 256 x 256 where as many can be made, all of dh's where
    # it has more, beside a piece of up to 256 MB
    for rows, dim, vocab in ((1024, 2048, 32000), (4096, 4096, 128256), (8192, 8192, 50257)):
        tiles = max(592, rows // 256 * (dim // 256))
        assert tiles * 2**18 < need(rows, dim, vocab) < tiles * 2**18 + (257 << 20) + rows * (2 * dim + 64)


def test_build_checks_the_registers_that_kernels_divide(tmp_path, monkeypatch) -> None:
    """A kernel that divides its launch's registers anew between its warps does not
    leave the build with another number of them."""
    spec = importlib.util.spec_from_file_location("cid_build_check",
                                                  ROOT / "cid-engine_b200" / "build.py")
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    name, registers, kernels = build._LAUNCH_REGISTERS["lm_head_int4.cu"]

    def log(used):
        lines = []
        for i in range(kernels):
            lines += [f"ptxas info : Compiling entry function '_Z{i}int4_head_kernelI6__halfLi16ELi1ELi2ELb0EE' "
                      "for 'sm_100a'", "ptxas info : Function properties", "    0 bytes stack frame",
                      f"ptxas info : Used {used if i == 3 else registers} registers, used 1 barriers",
                      f"ptxas info : Compiling entry function '_Z{i}int4_head_kernelI6__halfLi16ELi1ELi1ELb1EE'",
                      "ptxas info : Used 128 registers"]
        return "\n".join(lines)

    source, obj = tmp_path / "lm_head_int4.cu", tmp_path / "x.o"
    for used in (registers, registers - 8):
        obj.write_text("")
        monkeypatch.setattr(build, "_run", lambda cmd: log(used))
        assert build.launch_registers(log(used), name).count(registers) == kernels - (used != registers)
        if used == registers:
            build._compile_kernels(source, obj)
            assert obj.exists()
        else:
            with pytest.raises(SystemExit, match="96 registers"):
                build._compile_kernels(source, obj)
            assert not obj.exists()
