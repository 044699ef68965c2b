"""The residual and the gated RMS norm against their definitions in 64 bits."""
import ctypes
import sys
import threading

import pytest
import torch

from tests import _layer_ref as ref
from tests.conftest import state_rel_err

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
EPS = 1e-6
gpu = pytest.mark.gpu
WIDTHS = [1, 7, 8, 100, 128, 250, 256, 1000, 1024, 2048, 2056, 4096, 5333, 8192, 16384, 32761, 32767, 32768]


def rnd(*shape, dtype=torch.float32, device="cpu", scale=1.0, seed=0):
    gen = torch.Generator().manual_seed(seed + 7 * len(shape))
    return (torch.randn(shape, generator=gen) * scale).to(device, dtype)


def make(rows, width, dtype, dev, seed=0):
    return (rnd(rows, width, dtype=dtype, device=dev, seed=seed), rnd(rows, width, dtype=dtype, device=dev, scale=2.0, seed=seed + 1),
            1 + rnd(width, device=dev, scale=0.1, seed=seed + 2))


@gpu
@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_add_norm(pkg, cuda_dev, width, dtype):
    for rows in (1, 5):
        x, res, w = make(rows, width, dtype, cuda_dev, seed=rows)
        y, r = pkg.norm.launch_add_norm(x, res, w, EPS)
        want_r, want_y = ref.add_norm(x, res, w, EPS)
        ref.close(r, *want_r, "r")
        ref.close(y, *want_y, "y")
        y1, x1 = pkg.norm.launch_add_norm(x, None, w, EPS)
        assert x1 is x
        ref.close(y1, *ref.add_norm(x, None, w, EPS)[1], "y of x alone")


@gpu
@pytest.mark.parametrize("quant,width", [("row", w) for w in WIDTHS] + [("group", w) for w in WIDTHS if w % 128 == 0])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_add_norm_e4m3(pkg, cuda_dev, width, dtype, quant):
    x, res, w = make(6, width, dtype, cuda_dev)
    w[: width // 2] *= 1e-3  # groups of other magnitudes, codes among the subnormals
    res[3], x[3] = 0, 0
    q, r, s = pkg.norm.launch_add_norm(x, res, w, EPS, quant=quant)
    want_r, (y, err) = ref.add_norm(x, res, w, EPS)
    assert q.dtype == torch.float8_e4m3fn and s.shape == (6, 1 if quant == "row" else width // 128)
    ref.close(r, *want_r, "r")
    ref.codes_ok(q, s, y, err, width if quant == "row" else 128)
    assert not q[3].float().any() and bool((s[3] == torch.tensor(1e-12 / 448)).all())


@gpu
@pytest.mark.parametrize("rows", [0, 1, 3, 129, 2000])
@pytest.mark.parametrize("width", [64, 512, 2048, 4100])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_add_norm_backward(pkg, cuda_dev, rows, width, dtype):
    x, res, w = make(rows, width, dtype, cuda_dev)
    dy, dr = rnd(rows, width, dtype=dtype, device=cuda_dev, seed=8), rnd(rows, width, dtype=dtype, device=cuda_dev, seed=9)
    for d in (dr, None):
        dx, dw = pkg.norm.launch_add_norm_backward(dy, x, w, EPS, d_new_residual=d)
        want_dx, want_dw = ref.add_norm(None, None, w, EPS, dy=dy, dr=d, summed=x)
        ref.close(dx, *want_dx, "dx")
        ref.close(dw, *want_dw, "dweight")


@gpu
@pytest.mark.parametrize("width", [1, 7, 250, 1003, 5333])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_rows_of_odd_widths(pkg, cuda_dev, width, dtype):
    """More rows than the backward kernel has thread blocks, of widths where each row starts elsewhere in a
    16-byte vector: the results, and what lies beside the rows stays as it was.  The tensors begin off the boundary
    (the buffers' lengths are odd), on it and contiguous, and on it with 8 elements between rows; the last two are
    summed alike."""
    rows = 2003
    buf = rnd(4, rows * (width + 8), dtype=dtype, device=cuda_dev)
    x, res, dy, dr = (b.view(rows, width + 8)[:, :width] for b in buf)
    w = 1 + rnd(width, device=cuda_dev, scale=0.1)
    want_r, want_y = ref.add_norm(x, res, w, EPS)
    want_dx, want_dw = ref.add_norm(None, None, w, EPS, dy=dy, dr=dr, summed=x)
    n, out = rows * width, []
    whole = [t.contiguous() for t in (x, res, dy, dr)]
    apart = [torch.nn.functional.pad(t, (0, 8), value=9.0)[:, :width] for t in whole]
    for a, b, c, d in ((x, res, dy, dr), whole, apart):
        room = torch.full((3, (n + 71) // 8 * 8), 7.0, dtype=dtype, device=cuda_dev)
        codes = torch.full((n + 64,), 7.0, device=cuda_dev).to(torch.float8_e4m3fn)
        y, r, dx = (t[:n].view(rows, width) for t in room)
        pkg.norm.launch_add_norm(a, b, w, EPS, output=y, new_residual=r)
        q, _, scale = pkg.norm.launch_add_norm(a, b, w, EPS, quant="row", output=codes[:n].view(rows, width))
        _, dw = pkg.norm.launch_add_norm_backward(c, a, w, EPS, d_new_residual=d, dx=dx)
        ref.close(r, *want_r, "r")
        ref.close(y, *want_y, "y")
        ref.codes_ok(q, scale, *want_y, width)
        ref.close(dx, *want_dx, "dx")
        ref.close(dw, *want_dw, "dweight")
        assert bool((room[:, n:] == 7).all()) and bool((codes[n:].float() == 7).all())
        out.append([y.clone(), r.clone(), q.clone().float(), dx.clone(), dw])
    for t, u in zip(*out[1:]):
        assert torch.equal(t, u)


@gpu
@pytest.mark.parametrize("width", [8192, 20000, 32761, 32767, 32768])
def test_add_norm_backward_wide(pkg, cuda_dev, width):
    x, _, w = make(40, width, torch.bfloat16, cuda_dev)
    dy = rnd(40, width, dtype=torch.bfloat16, device=cuda_dev, seed=8)
    dx, dw = pkg.norm.launch_add_norm_backward(dy, x, w, EPS)
    want_dx, want_dw = ref.add_norm(None, None, w, EPS, dy=dy, summed=x)
    ref.close(dx, *want_dx, "dx")
    ref.close(dw, *want_dw, "dweight")


@gpu
@pytest.mark.parametrize("heads", [1, 3, 8, 32])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_gated_norm(pkg, cuda_dev, heads, dim, dtype):
    for tokens in (1, 37):
        x, z, dy = (rnd(tokens, heads, dim, dtype=dtype, device=cuda_dev, scale=2.0, seed=s) for s in (1, 2, 3))
        w = 1 + rnd(dim, device=cuda_dev, scale=0.1)
        y = pkg.norm.launch_gated_norm(x, z, w, EPS)
        want, err = ref.gated_norm(x, z, w, EPS)
        ref.close(y, want, err, "y")
        q, s = pkg.norm.launch_gated_norm(x, z, w, EPS, quant=True)
        assert s.shape == (tokens, heads)
        ref.codes_ok(q, s, want, err, dim)
        dx, dz, dw = pkg.norm.launch_gated_norm_backward(dy, x, z, w, EPS)
        want_dx, want_dz, want_dw = ref.gated_norm(x, z, w, EPS, dy=dy)
        ref.close(dx, *want_dx, "dx")
        ref.close(dz, *want_dz, "dz")
        ref.close(dw, *want_dw, "dweight")


@gpu
def test_gated_norm_many_tokens(pkg, cuda_dev):
    x, z, dy = (rnd(9001, 5, 128, dtype=torch.bfloat16, device=cuda_dev, seed=s) for s in (1, 2, 3))
    w = 1 + rnd(128, device=cuda_dev, scale=0.1)
    ref.close(pkg.norm.launch_gated_norm(x, z, w, EPS), *ref.gated_norm(x, z, w, EPS), "y")
    for g, want in zip(pkg.norm.launch_gated_norm_backward(dy, x, z, w, EPS), ref.gated_norm(x, z, w, EPS, dy=dy)):
        ref.close(g, *want)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_weights_of_the_inputs_type(pkg, cuda_dev, dtype):
    x, res, w = make(9, 520, dtype, cuda_dev)
    w16 = w.to(dtype)
    ref.close(pkg.norm.launch_add_norm(x, res, w16, EPS)[0], *ref.add_norm(x, res, w16, EPS)[1], "y")
    dx, dw = pkg.norm.launch_add_norm_backward(res, x, w16, EPS)
    want_dx, want_dw = ref.add_norm(None, None, w16, EPS, dy=res, summed=x)
    ref.close(dx, *want_dx, "dx")
    assert dw.dtype == torch.float32
    ref.close(dw, *want_dw, "dw")
    xh, zh, wh = x[:, :512].unflatten(1, (4, 128)), res[:, :512].unflatten(1, (4, 128)), w16[:128]
    ref.close(pkg.norm.launch_gated_norm(xh, zh, wh, EPS), *ref.gated_norm(xh, zh, wh, EPS), "gated")


@gpu
@pytest.mark.parametrize("off", [0, 8, 3])
def test_strided_and_unaligned_rows(pkg, cuda_dev, off):
    """Column blocks of a wider buffer.  Rows on 16-byte boundaries give the bits of contiguous ones;
    others are dealt to the threads, and so summed, in another order: the bounds hold, not the bits."""
    buf = rnd(11, 3000, dtype=torch.bfloat16, device=cuda_dev)
    x, res = buf[:, off:off + 1024], buf[:, off + 1024:off + 2048]
    w = 1 + rnd(1024, device=cuda_dev, scale=0.1)
    xc, resc = x.contiguous(), res.contiguous()
    xh, zh, wh = x.unflatten(1, (8, 128)), res.unflatten(1, (8, 128)), w[:128]

    def calls(x, res, xh, zh):
        n = pkg.norm
        return [n.launch_add_norm(x, res, w, EPS), n.launch_add_norm(x, res, w, EPS, quant="row"),
                n.launch_add_norm(x, res, w, EPS, quant="group"), n.launch_add_norm_backward(x, res, w, EPS, d_new_residual=x),
                (n.launch_gated_norm(xh, zh, wh, EPS),), n.launch_gated_norm_backward(zh, xh, zh, wh, EPS)]

    got = calls(x, res, xh, zh)
    if off % 8 == 0:
        for a, b in zip(got, calls(xc, resc, xc.unflatten(1, (8, 128)), resc.unflatten(1, (8, 128)))):
            for t, u in zip(a, b):
                assert torch.equal(t.float(), u.float())
    want_r, (y, err) = ref.add_norm(x, res, w, EPS)
    ref.close(got[0][0], y, err, "y")
    for k in range(3):
        ref.close(got[k][1], *want_r, "r")
    ref.codes_ok(got[1][0], got[1][2], y, err, 1024)
    ref.codes_ok(got[2][0], got[2][2], y, err, 128)
    for g, want in zip(got[3], ref.add_norm(None, None, w, EPS, dy=x, dr=x, summed=res)):
        ref.close(g, *want)
    ref.close(got[4][0], *ref.gated_norm(xh, zh, wh, EPS), "gated")
    for g, want in zip(got[5], ref.gated_norm(xh, zh, wh, EPS, dy=zh)):
        ref.close(g, *want)


@gpu
def test_offsets_past_32_bits(pkg, cuda_dev):
    big = torch.empty((40000, 65536), dtype=torch.bfloat16, device=cuda_dev)  # 2.6e9 elements
    x, z = big[:, -256:], rnd(40000, 256, dtype=torch.bfloat16, device=cuda_dev)
    x.copy_(rnd(40000, 256, dtype=torch.bfloat16, device=cuda_dev, seed=1))
    w = 1 + rnd(256, device=cuda_dev, scale=0.1)
    assert torch.equal(pkg.norm.launch_add_norm(x, z, w, EPS)[0], pkg.norm.launch_add_norm(x.contiguous(), z, w, EPS)[0])
    xh, zh = x.unflatten(1, (2, 128)), z.unflatten(1, (2, 128))
    assert torch.equal(pkg.norm.launch_gated_norm(xh, zh, w[:128], EPS), pkg.norm.launch_gated_norm(xh.contiguous(), zh, w[:128], EPS))


@gpu
@pytest.mark.parametrize("width", [17, 250, 1003, 5333])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_rows_of_odd_widths_do_not_leak(pkg, cuda_dev, bad, width):
    """A vector of 8 elements can hold the end of one row and the start of the next; in place too."""
    x, res, w = make(40, width, torch.bfloat16, cuda_dev)
    dy = rnd(40, width, dtype=torch.bfloat16, device=cuda_dev, seed=8)
    keep = torch.arange(40, device=cuda_dev) % 3 != 1
    x2, dy2 = x.clone(), dy.clone()
    x2[~keep], dy2[~keep] = bad, bad
    for quant in (None, "row"):
        good, got = (pkg.norm.launch_add_norm(t, res.clone(), w, EPS, quant=quant) for t in (x, x2))
        in_place = x2.clone()
        again = pkg.norm.launch_add_norm(in_place, res, w, EPS, quant=quant, new_residual=in_place)
        for a, b, c in zip(good, got, again):
            assert torch.equal(a[keep].float(), b[keep].float()) and torch.equal(a[keep].float(), c[keep].float())
        assert bool(got[0][~keep].float().isnan().all())
    dx, dx2 = (pkg.norm.launch_add_norm_backward(g, t, w, EPS, d_new_residual=g)[0] for g, t in ((dy, x), (dy2, x2)))
    assert torch.equal(dx[keep], dx2[keep]) and bool(dx2[~keep].isnan().all())


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_weights_of_odd_widths(pkg, cuda_dev, dtype):
    """Weights of either type that begin on a 16-byte boundary and off it."""
    x, res, w = make(9, 1003, dtype, cuda_dev)
    for wt in (w, w.to(dtype)):
        off = torch.cat([wt[:1], wt])[1:]
        for weight in (wt, off):
            ref.close(pkg.norm.launch_add_norm(x, res, weight, EPS)[0], *ref.add_norm(x, res, wt, EPS)[1], "y")
            dx, dw = pkg.norm.launch_add_norm_backward(res, x, weight, EPS)
            want_dx, want_dw = ref.add_norm(None, None, wt, EPS, dy=res, summed=x)
            ref.close(dx, *want_dx, "dx")
            ref.close(dw, *want_dw, "dw")


@gpu
def test_in_place(pkg, cuda_dev):
    x, res, w = make(33, 2048, torch.bfloat16, cuda_dev)
    y, r = pkg.norm.launch_add_norm(x, res, w, EPS)
    for target in (res.clone(), x.clone()):
        other = x if torch.equal(target, res) else res
        y2, r2 = pkg.norm.launch_add_norm(other, target, w, EPS, new_residual=target)
        assert r2 is target and torch.equal(y2, y) and torch.equal(r2, r)
    xh, zh = x.unflatten(1, (16, 128)).contiguous(), res.unflatten(1, (16, 128))
    want = pkg.norm.launch_gated_norm(xh, zh, w[:128], EPS)
    got = pkg.norm.launch_gated_norm(xh, zh, w[:128], EPS, output=xh)
    assert got is xh and torch.equal(got, want)


@gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_rows_do_not_leak(pkg, cuda_dev, bad):
    """A NaN (or infinity) spoils its own row, group or head, and its scale says so."""
    x, res, w = make(40, 1024, torch.bfloat16, cuda_dev)
    x2 = x.clone()
    x2[7, 300] = bad
    keep = torch.arange(40, device=cuda_dev) != 7
    for quant in (None, "row", "group"):
        good, got = (pkg.norm.launch_add_norm(t, res, w, EPS, quant=quant) for t in (x, x2))
        for a, b in zip(good, got):
            assert torch.equal(a[keep].float(), b[keep].float())
        assert bool(got[0][7, 300].float().isnan())
        if quant == "row":
            assert bool(got[2][7].isnan().all())
        if quant == "group":
            assert bool(got[2][7, 300 // 128].isnan())
    xh, x2h, zh = (t.unflatten(1, (8, 128)) for t in (x, x2, res))
    (q, s), (q2, s2) = (pkg.norm.launch_gated_norm(t, zh, w[:128], EPS, quant=True) for t in (xh, x2h))
    mask = torch.ones(40, 8, dtype=torch.bool, device=cuda_dev)
    mask[7, 300 // 128] = False
    assert torch.equal(q[mask].float(), q2[mask].float()) and torch.equal(s[mask], s2[mask]) and bool(s2[~mask].isnan().all())


@gpu
def test_large_and_tiny_values(pkg, cuda_dev):
    """fp16 sums beyond its range, gates far out, subnormal rows."""
    x = torch.full((3, 256), 60000.0, dtype=torch.float16, device=cuda_dev)
    w = torch.ones(256, device=cuda_dev)
    y, r = pkg.norm.launch_add_norm(x, x, w, EPS)
    assert bool(r.isinf().all())  # 120000 does not fit, the norm of the unrounded sum does
    ref.close(y, *ref.add_norm(x, x, w, EPS)[1], "y")
    x = rnd(4, 2, 128, device=cuda_dev) * 1e-20
    z = rnd(4, 2, 128, device=cuda_dev) * 60
    z[0, 0, 0], z[0, 0, 1] = 1e4, -1e4
    ref.close(pkg.norm.launch_gated_norm(x, z, w[:128], EPS), *ref.gated_norm(x, z, w[:128], EPS), "y")


@gpu
def test_reproducible_streams_and_graphs(pkg, cuda_dev):
    x, res, w = make(3000, 1024, torch.bfloat16, cuda_dev)
    first = pkg.norm.launch_add_norm_backward(res, x, w, EPS, d_new_residual=res)
    xh, zh = x.unflatten(1, (8, 128)), res.unflatten(1, (8, 128))
    first_g = pkg.norm.launch_gated_norm_backward(zh, xh, zh, w[:128], EPS)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(cuda_dev) for _ in range(2)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append((pkg.norm.launch_add_norm_backward(res, x, w, EPS, d_new_residual=res),
                        pkg.norm.launch_gated_norm_backward(zh, xh, zh, w[:128], EPS)))
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append((pkg.norm.launch_add_norm_backward(res, x, w, EPS, d_new_residual=res),
                         pkg.norm.launch_gated_norm_backward(zh, xh, zh, w[:128], EPS)))
        graphs.append(g)
    for g in graphs + graphs[::-1]:
        g.replay()
    torch.cuda.synchronize()
    for a, b in got + outs:
        for t, u in zip(a + b, first + first_g):
            assert torch.equal(t, u)


@gpu
def test_autograd(pkg, cuda_dev):
    x, res, w = make(50, 256, torch.float32, cuda_dev)
    dy, dr = rnd(50, 256, device=cuda_dev, seed=8), rnd(50, 256, device=cuda_dev, seed=9)
    lx, lr, lw = (t.clone().requires_grad_() for t in (x, res, w))
    y, r = pkg.norm.add_norm(lx, lr, lw, EPS)
    ((y * dy).sum() + (r * dr).sum()).backward()
    dx, dw = pkg.norm.launch_add_norm_backward(dy, r.detach(), w, EPS, d_new_residual=dr)
    assert torch.equal(lx.grad, dx) and torch.equal(lr.grad, dx) and torch.equal(lw.grad, dw)
    x64, r64, w64 = (t.double().requires_grad_() for t in (x, res, w))
    s = x64 + r64
    ((s / (s.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * w64 * dy).sum() + (s * dr).sum()).backward()
    want_dx, want_dw = ref.add_norm(None, None, w, EPS, dy=dy, dr=dr, summed=x.double() + res.double())
    assert torch.allclose(x64.grad, want_dx[0]) and torch.allclose(w64.grad, want_dw[0])  # the formulas are the gradients
    lx.grad = None
    y, same = pkg.norm.add_norm(lx, None, w, EPS)
    assert same is lx
    (y * dy).sum().backward()
    assert torch.equal(lx.grad, pkg.norm.launch_add_norm_backward(dy, x, w, EPS)[0])

    xh, zh, dyh = (t.unflatten(1, (2, 128)) for t in (x, res, dy))
    leaves = [t.clone().requires_grad_() for t in (xh, zh, w[:128])]
    (pkg.norm.gated_norm(*leaves, EPS) * dyh).sum().backward()
    for leaf, want in zip(leaves, pkg.norm.launch_gated_norm_backward(dyh, xh, zh, w[:128], EPS)):
        assert torch.equal(leaf.grad, want)
    x64, z64, w64 = (t.double().requires_grad_() for t in (xh, zh, w[:128]))
    (x64 / (x64.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * w64 * torch.nn.functional.silu(z64) * dyh).sum().backward()
    for leaf, want in zip((x64, z64, w64), ref.gated_norm(xh, zh, w[:128], EPS, dy=dyh)):
        assert torch.allclose(leaf.grad, want[0])


# --------------------------------------------------- as the paths call them --
@gpu
@pytest.mark.parametrize("quant", [False, True])
def test_launch_gdn_with_out_norm(pkg, cuda_dev, quant):
    """decode and prefill with out_norm: the plain call's output, normed."""
    w = 1 + rnd(128, device=cuda_dev, scale=0.1)
    dec = pkg.inputs.make_decode_inputs(5, seed=1).to(cuda_dev)
    tok = pkg.inputs.make_decode_inputs(5, seed=1, tokens=3).to(cuda_dev)
    pre = pkg.inputs.make_prefill_inputs([70, 0, 200], seed=2).to(cuda_dev)
    for launch, inp in ((pkg.decode.launch_gdn, dec), (pkg.decode.launch_gdn, tok), (pkg.prefill.launch_gdn, pre)):
        plain, plain_state = launch(*inp.args())
        z = rnd(*plain.shape, dtype=torch.bfloat16, device=cuda_dev, seed=3)
        norm = pkg.norm.OutputNorm(z, w)
        if quant:
            norm.codes = torch.empty(plain.shape, dtype=torch.float8_e4m3fn, device=cuda_dev)
            norm.scale = torch.empty(plain.shape[:-1], dtype=torch.float32, device=cuda_dev)
        out, state = launch(*inp.args(), out_norm=norm)
        assert torch.equal(state, plain_state)
        want, err = ref.gated_norm(plain, z, w, 1e-6)
        if quant:
            assert torch.equal(out, plain)
            ref.codes_ok(norm.codes, norm.scale, want, err, 128)
        else:
            ref.close(out, want, err, "normed output")
    with pytest.raises(ValueError, match="z must have"):
        pkg.decode.launch_gdn(*dec.args(), out_norm=pkg.norm.OutputNorm(z, w))
    with pytest.raises(ValueError, match="go together"):
        pkg.decode.launch_gdn(*dec.args(), out_norm=pkg.norm.OutputNorm(dec.v, w, codes=z))


@gpu
def test_a_layer_of_them(pkg, cuda_dev):
    """Residual norm, a projection, both recurrences, the gated norm, a projection back: as a model would
    run them, prompt then tokens, against the same layer on the whole sequence."""
    width, C, T = 512, 256, 90
    gen = torch.Generator().manual_seed(0)
    p = lambda *s: (torch.randn(s, generator=gen) / s[0] ** 0.5).to(cuda_dev)  # noqa: E731
    w_in, w_out, w1, w2 = p(width, 4 * C), p(C, width), 1 + p(width) * 0.1, 1 + p(128) * 0.1
    A_log, dt_bias = torch.rand(C, generator=gen).to(cuda_dev), -2 * torch.ones(C, device=cuda_dev)
    x, res = (torch.randn(T, width, generator=gen).to(cuda_dev) for _ in range(2))

    def layer(x, res, recur):
        y, r = pkg.norm.launch_add_norm(x, res, w1)
        proj = y @ w_in
        xs, a, b, z = proj.split(C, dim=1)
        h = recur(xs, A_log, a, dt_bias, b)
        o = pkg.norm.launch_gated_norm(h.unflatten(1, (2, 128)), z.unflatten(1, (2, 128)), w2)
        return o.flatten(1) @ w_out, r

    s = {}

    def scan(n):
        def run(*g):
            y, s["h"] = pkg.recurrence.launch_scan(*g, torch.tensor([0, n]))
            return y
        return run

    def step(*g):
        return pkg.recurrence.launch_step(*g, s["h"], new_state=s["h"])[0]

    whole, _ = layer(x, res, scan(T))
    last = s["h"]
    parts = [layer(x[:80], res[:80], scan(80))[0]] + [layer(x[t:t + 1], res[t:t + 1], step)[0] for t in range(80, T)]
    # the two runs differ by the fp32 products' blocking: 512- and 256-term sums, 2^-24 sqrt(512) each, and the layer's gain
    assert state_rel_err(torch.cat(parts), whole) < 1e-4 and state_rel_err(s["h"], last) < 1e-4


# ---------------------------------------------------------------- refusals --
@gpu
def test_refusals(pkg, cuda_dev):
    n = pkg.norm
    x, res, w = make(4, 256, torch.bfloat16, cuda_dev)
    for match, args, kw in [
            ("x must be a", (x[0], res, w), {}), ("bfloat16, float16 or float32", (x.double(), res, w), {}),
            ("residual must be", (x, res.float(), w), {}), ("residual must have shape", (x, res[:2], w), {}),
            ("contiguous rows", (x.t().contiguous().t(), res, w), {}), ("overlapping rows", (x[:1].expand(4, 256), res, w), {}),
            ("weight must have shape", (x, res, w[:5]), {}), ("weight must be float32", (x, res, w.double()), {}),
            ("quant must be", (x, res, w), {"quant": "column"}), ("multiple of 128", (x[:, :200], res[:, :200], w[:200]), {"quant": "group"}),
            ("eps", (x, res, w, -1.0), {}), ("needs a residual", (x, None, w), {"new_residual": res}),
            ("scale needs quant", (x, res, w), {"scale": w}), ("output must be", (x, res, w), {"output": x, "quant": "row"}),
            ("scale must have shape", (x, res, w), {"scale": w, "quant": "row"}), ("new_residual must be contiguous", (x, res, w), {"new_residual": torch.cat([res, res], 1)[:, :256]})]:
        with pytest.raises(ValueError, match=match):
            n.launch_add_norm(*args, **kw)
    xh, zh, wh = x.unflatten(1, (2, 128)), res.unflatten(1, (2, 128)), w[:128]
    for match, args, kw in [
            ("tokens, heads, dim", (x, res, wh), {}), ("z must have", (xh, zh[:2], wh), {}),
            ("head dim must be", (xh.reshape(4, 8, 32), zh.reshape(4, 8, 32), wh[:32]), {}), ("weight must have shape", (xh, zh, w), {}),
            ("contiguous heads", (xh.transpose(1, 2).contiguous().transpose(1, 2), zh, wh), {}), ("scale needs quant", (xh, zh, wh), {"scale": w}),
            ("output must not be z", (xh, zh, wh), {"output": zh}), ("output must be", (xh, zh, wh), {"output": xh, "quant": True})]:
        with pytest.raises(ValueError, match=match):
            n.launch_gated_norm(*args, **kw)
    with pytest.raises(ValueError, match="d_output must"):
        n.launch_add_norm_backward(res[:2], x, w)
    with pytest.raises(ValueError, match="d_output must"):
        n.launch_gated_norm_backward(zh[:2], xh, zh, wh)
    out = torch.empty_like(x)
    with pytest.raises(ValueError, match="output must not be new_residual"):
        n.launch_add_norm(x, res, w, output=out, new_residual=out)
    with pytest.raises(ValueError, match="dz must not be dx"):
        n.launch_gated_norm_backward(zh, xh, zh, wh, dx=out.view_as(xh), dz=out.view_as(xh))


def test_cpu_tensors_are_refused(pkg):
    x, res, w = make(4, 256, torch.bfloat16, "cpu")
    with pytest.raises(ValueError, match="CUDA tensor"):
        pkg.norm.launch_add_norm(x, res, w)
    with pytest.raises(ValueError, match="CUDA tensor"):
        pkg.norm.launch_add_norm_backward(x, res, w)
    with pytest.raises(ValueError, match="CUDA tensor"):
        pkg.norm.launch_gated_norm(x.unflatten(1, (2, 128)), res.unflatten(1, (2, 128)), w[:128])


def test_capi_refusals(pkg):
    """Host-side checks come before any device call, so they answer without a GPU."""
    lib, C = pkg._capi.load(), pkg._capi
    buf = ctypes.create_string_buffer(8192)
    p = (ctypes.addressof(buf) + 63) // 64 * 64

    def put(s, kw):
        for k, v in kw.items():
            setattr(s, k, v)
        return ctypes.byref(s)

    def add(**kw):
        return put(C.GdnAddNormArgs(p, p, 256, 256, p, C.DTYPE_F32, C.DTYPE_BF16, 0, EPS, 2, 256, p, p, p), kw)

    def gated(**kw):
        return put(C.GdnGatedNormArgs(p, p, 256, 256, p, C.DTYPE_F32, C.DTYPE_BF16, 0, EPS, 2, 2, 128, p, p), kw)

    def grad(**kw):
        return put(C.GdnNormGradArgs(p, 256, None, 0, p, p, p), kw)

    NULL, SIZE, ALIGN, WS, DTYPE = 1, 2, 3, 4, 6
    for want, kw in [(NULL, dict(x=None)), (NULL, dict(weight=None)), (NULL, dict(output=None)), (NULL, dict(new_residual=None)),
                     (NULL, dict(quant=1, scale=None)), (SIZE, dict(rows=-1)), (SIZE, dict(width=0)), (SIZE, dict(width=40000)),
                     (SIZE, dict(quant=3)), (SIZE, dict(quant=2, width=200)), (SIZE, dict(x_stride=255)), (SIZE, dict(eps=-1.0)),
                     (ALIGN, dict(x=p + 1)), (ALIGN, dict(weight=p + 2)), (DTYPE, dict(dtype=9)), (DTYPE, dict(weight_dtype=1))]:
        assert lib.gdn_add_norm_launch(add(**kw), None) == want, kw
    for want, kw in [(NULL, dict(z=None)), (NULL, dict(output=None)), (SIZE, dict(head_dim=96)), (SIZE, dict(heads=0)),
                     (SIZE, dict(tokens=1 << 31)), (SIZE, dict(quant=1)), (SIZE, dict(z_stride=3)), (ALIGN, dict(z=p + 1)),
                     (DTYPE, dict(dtype=-1))]:
        assert lib.gdn_gated_norm_launch(gated(**kw), None) == want, kw
    for fn, args, need in ((lib.gdn_add_norm_backward_launch, add, lib.gdn_add_norm_backward_workspace_size(2, 256)),
                           (lib.gdn_gated_norm_backward_launch, gated, lib.gdn_gated_norm_backward_workspace_size(2, 2, 128))):
        assert need > 0
        assert fn(args(), grad(dx=None), p, need, None) == NULL
        assert fn(args(), grad(d_weight=None), p, need, None) == NULL
        assert fn(args(), grad(d_output_stride=1), p, need, None) == SIZE
        assert fn(args(quant=2), grad(), p, need, None) == SIZE
        assert fn(args(), grad(dx=p + 1), p, need, None) == ALIGN
        assert fn(args(), grad(), p, need - 1, None) == WS
        assert fn(args(), grad(), None, need, None) == WS
    assert lib.gdn_add_norm_launch(None, None) == NULL and lib.gdn_gated_norm_launch(None, None) == NULL


# ------------------------------------------------------- codes of a quotient --
def _e4m3_of(y, scale):
    """The codes by definition: torch's own fp32 division by the stored scales, then its conversion."""
    return (y / scale[..., None]).clamp(-448, 448).to(torch.float8_e4m3fn).float()


def _scale_of(y):
    # a tensor, since by a number torch multiplies with its reciprocal
    return y.abs().amax(-1).clamp(min=1e-12) / torch.full((), 448.0, device=y.device)


@gpu
@pytest.mark.parametrize("quant,width", [("row", 4096), ("group", 4096), ("row", 1003), ("row", 250)])
def test_codes_are_y_over_the_stored_scale(pkg, cuda_dev, quant, width):
    """Every code of 33 million, at its ties too.  An fp32 output is the y that the codes are made of."""
    x, res, w = make((1 << 25) // width, width, torch.float32, cuda_dev)
    y, _ = pkg.norm.launch_add_norm(x, res, w, EPS)
    q, _, s = pkg.norm.launch_add_norm(x, res, w, EPS, quant=quant)
    per = y.unflatten(1, (s.shape[1], -1))
    assert torch.equal(s, _scale_of(per))
    assert torch.equal(q.float(), _e4m3_of(per, s).flatten(1))


@gpu
def test_gated_codes_are_y_over_the_stored_scale(pkg, cuda_dev):
    x, z = (rnd(65536, 4, 128, device=cuda_dev, seed=k) for k in (1, 2))
    w = 1 + rnd(128, device=cuda_dev, scale=0.1)
    y = pkg.norm.launch_gated_norm(x, z, w, EPS)
    q, s = pkg.norm.launch_gated_norm(x, z, w, EPS, quant=True)
    assert torch.equal(s, _scale_of(y)) and torch.equal(q.float(), _e4m3_of(y, s))


@gpu
@pytest.mark.parametrize("quant", ["row", "group"])
def test_codes_beside_an_infinite_output(pkg, cuda_dev, quant):
    """A weight that overflows its column: that code is NaN, its neighbours' are 0 over an infinite scale; the
    smallest and the largest finite scales hold too."""
    x, res, w = make(5, 256, torch.float32, cuda_dev)
    w[3] = 3e38
    x[:, 3], res[:, 3] = 4.0, 4.0
    q, _, s = pkg.norm.launch_add_norm(x, res, w, EPS, quant=quant)
    assert bool(s[:, 0].isinf().all()) and bool(q[:, 3].float().isnan().all())
    near = q[:, :128].float()
    near[:, 3] = 0
    assert not near.any()
    for big in (1e-30, 1e-13, 1e-12, 3e36, 3e37):
        v = rnd(256, device=cuda_dev).sign() * big
        y, _ = pkg.norm.launch_add_norm(x[:, :], None, v, EPS)
        q, _, s = pkg.norm.launch_add_norm(x, None, v, EPS, quant=quant)
        per = y.unflatten(1, (s.shape[1], -1))
        assert torch.equal(s, _scale_of(per)) and torch.equal(q.float(), _e4m3_of(per, s).flatten(1))


@gpu
@pytest.mark.parametrize("off", [0, 1])
def test_norms_of_nothing(pkg, cuda_dev, off):
    """No tokens or rows, with weights on a 16-byte boundary and off it: zeros, and nothing is read."""
    n, w = pkg.norm, torch.ones(129, device=cuda_dev)[off:off + 128]
    e = torch.empty(0, 3, 128, dtype=torch.bfloat16, device=cuda_dev)
    dx, dz, dw = n.launch_gated_norm_backward(e, e, e, w, EPS)
    assert dx.shape == dz.shape == e.shape and not dw.any()
    assert n.launch_gated_norm(e, e, w, EPS).shape == e.shape
    q, s = n.launch_gated_norm(e, e, w, EPS, quant=True)
    assert q.shape == e.shape and s.shape == (0, 3)
    r = e[:, 0]
    dx, dw = n.launch_add_norm_backward(r, r, w, EPS, d_new_residual=r)
    assert dx.shape == r.shape and not dw.any()
    for quant in (None, "row", "group"):
        assert n.launch_add_norm(r, r, w, EPS, quant=quant)[0].shape == r.shape
    assert pkg.prefill.device_status(cuda_dev) == 0


def test_backward_waits_for_its_copies(pkg):
    """A wait that runs out is not forced on a GPU; that the kernel then waits for every copy under way is held here:
    the stage and phase that it waits for, for the rows that were asked for, are those of the main loop."""
    source = (pkg._build.CSRC / "gdn_norm.cu").read_text()
    body = source[source.index("gdn_add_norm_backward_kernel(const NormParams p"):]
    body = body[:body.index("\n}\n")]
    give_up = body[body.index("if (!tc05::mbar_wait(bar + 8 * stage, phase)) {"):body.index("return record_status")]
    assert "(stage + i) % p.stages" in give_up and "phase ^ (at < stage)" in give_up and "< p.rows" in give_up
    for stages in (2, 3):
        for first in range(8):  # rows `first` .. of this block: the main loop's stage and phase of each
            stage, phase, seen = 0, 0, []
            for _ in range(first + stages):
                seen.append((stage, phase))
                stage = 0 if stage + 1 == stages else stage + 1
                phase ^= stage == 0
            at, ph = seen[first]
            want = seen[first:first + stages]
            assert [((at + i) % stages, ph ^ ((at + i) % stages < at)) for i in range(stages)] == want


@gpu
def test_backward_from_four_threads(pkg, cuda_dev):
    """Host threads with a stream each, at two widths whose rows take different amounts of one kernel's shared memory;
    then both widths in one graph.  Packed arguments, so that the threads spend their time inside the library."""
    lib, C, rows = pkg._capi.load(), pkg._capi, 8
    refused, calls, results = [], [], []
    for k, width in enumerate((4096, 8192, 4096, 8192)):
        x, _, w = make(rows, width, torch.bfloat16, cuda_dev, seed=k)
        dy = rnd(rows, width, dtype=torch.bfloat16, device=cuda_dev, seed=8)
        need = int(lib.gdn_add_norm_backward_workspace_size(rows, width))
        t = [x, dy, w, torch.empty_like(x), torch.empty_like(w), torch.empty(need, dtype=torch.uint8, device=cuda_dev),
             torch.cuda.Stream(cuda_dev)]
        args = pkg.norm._pack_add(x.data_ptr(), 0, width, 0, w.data_ptr(), C.DTYPE_F32, C.DTYPE_BF16, 0, EPS, rows, width, 0, 0, 0)
        grads = pkg.norm._pack_grad(dy.data_ptr(), width, 0, 0, t[3].data_ptr(), 0, t[4].data_ptr())
        calls.append((args, grads, t[5].data_ptr(), need, t[6].cuda_stream))
        results.append(t)
    torch.cuda.synchronize()

    def work(call):
        torch.cuda.set_device(cuda_dev)
        refused.extend(rc for rc in (lib.gdn_add_norm_backward_launch(*call) for _ in range(10000)) if rc)

    interval = sys.getswitchinterval()
    sys.setswitchinterval(1e-6)
    try:
        threads = [threading.Thread(target=work, args=(c,)) for c in calls]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
    finally:
        sys.setswitchinterval(interval)
    torch.cuda.synchronize()
    assert not refused
    for x, dy, w, dx, dw, *_ in results:
        want_dx, want_dw = ref.add_norm(None, None, w, EPS, dy=dy, summed=x)
        ref.close(dx, *want_dx, "dx")
        ref.close(dw, *want_dw, "dweight")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        captured = [pkg.norm.launch_add_norm_backward(t[1], t[0], t[2], EPS) for t in results[:2]]
    g.replay()
    torch.cuda.synchronize()
    for (dx, dw), t in zip(captured, results):
        assert torch.equal(dx, t[3]) and torch.equal(dw, t[4])


# ----------------------------------------------- sums with one term to them --
@gpu
def test_gated_weight_gradient_of_one_head(pkg, cuda_dev):
    """d_output in one head of many: the weight's gradient is that head's term, wherever it lies in the blocks' turns
    (1184 blocks of 16 heads) and in the last, partial one."""
    tokens, heads, dim = 9001, 5, 128
    x, z, dy = (rnd(tokens, heads, dim, dtype=torch.bfloat16, device=cuda_dev, seed=s) for s in (1, 2, 3))
    w = 1 + rnd(dim, device=cuda_dev, scale=0.1)
    n = tokens * heads
    for item in (0, 15, 16, 18943, 18944, 37887, 37888, 37888 + 7100, n - 6, n - 5, n - 1):
        one = torch.zeros_like(dy).view(n, dim)
        one[item] = dy.view(n, dim)[item]
        dw = pkg.norm.launch_gated_norm_backward(one.view_as(dy), x, z, w, EPS)[2]
        at = tuple(t.view(n, 1, dim)[item:item + 1] for t in (x, z, dy))
        want, err = ref.gated_norm(*at[:2], w, EPS, dy=at[2])[2]
        ref.close(dw, want, err, f"head {item}")


@gpu
@pytest.mark.parametrize("width", [250, 1003, 4096])
def test_weight_gradient_of_one_row(pkg, cuda_dev, width):
    rows = 2003
    x, _, w = make(rows, width, torch.bfloat16, cuda_dev)
    dy = rnd(rows, width, dtype=torch.bfloat16, device=cuda_dev, seed=8)
    for row in (0, 1, 143, 144, 147, 148, 295, 296, 1183, 1184, 1999, 2000, 2002):
        one = torch.zeros_like(dy)
        one[row] = dy[row]
        dw = pkg.norm.launch_add_norm_backward(one, x, w, EPS)[1]
        want, err = ref.add_norm(None, None, w, EPS, dy=dy[row:row + 1], summed=x[row:row + 1])[1]
        ref.close(dw, want, err, f"row {row}")
