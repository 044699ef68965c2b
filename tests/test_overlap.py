"""Outputs that share memory with an input or another output are refused; an output that is an input is not."""
import ctypes
import random
import subprocess

import pytest
import torch

from tests.test_norm import EPS, make, rnd
from tests.test_recurrence import backward, gates
from tests.test_recurrence import make as make_scan

gpu = pytest.mark.gpu


@pytest.fixture(scope="module")
def meet(pkg, tmp_path_factory):
    """``meet((p, rows, step, width), (...))`` of the library's host code, in bytes."""
    tmp = tmp_path_factory.mktemp("overlap")
    (tmp / "shim.cpp").write_text(
        '#include "gdn_overlap.cuh"\n'
        'extern "C" int meet(const int64_t* a, const int64_t* b) {\n'
        '    return gdn::rows_meet({(const void*)a[0], a[1], a[2], a[3]}, {(const void*)b[0], b[1], b[2], b[3]});\n}\n')
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", f"-I{pkg._build.CSRC}", "-o", tmp / "shim.so", tmp / "shim.cpp"], check=True)
    fn = ctypes.CDLL(str(tmp / "shim.so")).meet
    row = ctypes.c_int64 * 4
    return lambda a, b: bool(fn(row(*a), row(*b)))


def _bytes(p, rows, step, width):
    return {p + r * step + k for r in range(rows) for k in range(width)}


def test_rows_meet(meet):
    """Against the sets of bytes: exact where the steps are equal or one tensor is contiguous, else never too late."""
    rng = random.Random(0)
    refused = 0
    for _ in range(20000):
        step = rng.randint(1, 24)
        a, b = ((rng.randint(1, 120), rng.randint(1, 6), s, rng.randint(1, s))
                for s in (step, step if rng.random() < 0.6 else rng.randint(1, 24)))
        truth = bool(_bytes(*a) & _bytes(*b))
        got = meet(a, b)
        assert got == meet(b, a)
        if a[2] == b[2] or 1 in (a[1], b[1]) or a[2] == a[3] or b[2] == b[3]:
            assert got == truth, (a, b)
        else:
            assert got or not truth, (a, b)
            refused += got and not truth
    assert refused < 3000
    assert not meet((0, 3, 4, 4), (0, 3, 4, 4)) and not meet((8, 0, 4, 4), (8, 3, 4, 4))  # absent or empty
    big = 1 << 40  # past 32 bits: two column blocks, and the same one row apart
    assert not meet((big, 1 << 21, 1 << 20, 512), (big + 512, 1 << 21, 1 << 20, 512))
    assert meet((big, 1 << 21, 1 << 20, 512), (big + (1 << 40) + 511, 1 << 21, 1 << 20, 512))


def test_capi_refuses_overlaps(pkg):
    """Only calls that are refused: the host's checks answer without a device."""
    lib, C = pkg._capi.load(), pkg._capi
    buf = ctypes.create_string_buffer(1 << 16)
    p = (ctypes.addressof(buf) + 4095) // 4096 * 4096
    at = [p + 1024 * k for k in range(20)]

    def scan(**kw):
        a = C.GdnScanArgs(at[0], at[1], at[2], 16, 16, 16, at[3], at[4], at[5], at[6], C.GDN_SEQLENS_INT64, C.DTYPE_BF16, 4, 2, 16,
                          at[7], 16, at[8], at[9])
        for k, v in kw.items():
            setattr(a, k, v)
        return ctypes.byref(a)

    OVER = C.GDN_ERR_OVERLAP
    for kw in [dict(output=at[0] + 2), dict(output=at[1] + 64), dict(output=at[2]), dict(output=at[5] + 4), dict(new_state=at[5] + 64),
               dict(new_state=at[6] + 16), dict(checkpoints=at[8] + 64), dict(checkpoints=at[0]), dict(output=at[9] - 64)]:
        assert lib.gdn_scan_launch(scan(**kw), None) == OVER, kw

    def grads(**kw):
        g = C.GdnScanGradArgs(at[10], 16, at[11], at[12], at[13], at[14], 16, 16, 16, at[15], at[16], at[17])
        for k, v in kw.items():
            setattr(g, k, v)
        return ctypes.byref(g)

    for kw in [dict(dx=at[0]), dict(dx=at[13] + 32), dict(da=at[10] + 2), dict(db=at[9]), dict(d_state=at[11]), dict(dA_log=at[16] + 8)]:
        assert lib.gdn_scan_backward_launch(scan(), grads(**kw), None) == OVER, kw
    step = dict(num_seqs=4, checkpoints=None)
    for kw in [dict(output=at[0] + 2), dict(new_state=at[5] + 4), dict(output=at[8] + 16)]:
        assert lib.gdn_scan_step_launch(scan(**step, **kw), 1, None) == OVER, kw

    def add(**kw):
        a = C.GdnAddNormArgs(at[0], at[1], 256, 256, at[2], C.DTYPE_F32, C.DTYPE_BF16, 0, EPS, 2, 256, at[4], at[6], at[8])
        for k, v in kw.items():
            setattr(a, k, v)
        return ctypes.byref(a)

    for kw in [dict(output=at[0] + 16), dict(new_residual=at[1] + 2), dict(output=at[6]), dict(output=at[0], quant=1), dict(scale=at[4], quant=1),
               dict(output=at[2] + 512), dict(output=at[0], x_stride=264), dict(new_residual=at[0], x_stride=300)]:
        assert lib.gdn_add_norm_launch(add(**kw), None) == OVER, kw

    def gated(**kw):
        a = C.GdnGatedNormArgs(at[0], at[1], 256, 256, at[2], C.DTYPE_F32, C.DTYPE_BF16, 0, EPS, 2, 2, 128, at[4], at[8])
        for k, v in kw.items():
            setattr(a, k, v)
        return ctypes.byref(a)

    for kw in [dict(output=at[0] + 256), dict(output=at[1], quant=2), dict(scale=at[4] + 8, quant=2), dict(output=at[0], x_stride=512)]:
        assert lib.gdn_gated_norm_launch(gated(**kw), None) == OVER, kw

    def grad(**kw):
        g = C.GdnNormGradArgs(at[10], 256, None, 0, at[12], at[13], at[14])
        for k, v in kw.items():
            setattr(g, k, v)
        return ctypes.byref(g)

    for fn, args, need in ((lib.gdn_add_norm_backward_launch, add, lib.gdn_add_norm_backward_workspace_size(2, 256)),
                           (lib.gdn_gated_norm_backward_launch, gated, lib.gdn_gated_norm_backward_workspace_size(2, 2, 128))):
        for kw in [dict(dx=at[10] + 16), dict(dx=at[0] + 16), dict(d_weight=at[2]), dict(d_weight=at[12] + 16)]:
            assert fn(args(), grad(**kw), at[15], need, None) == OVER, kw
        assert fn(args(), grad(), at[12], need, None) == OVER
    assert lib.gdn_gated_norm_backward_launch(gated(), grad(dz=at[12] + 64), at[15], need, None) == OVER


@gpu
def test_scan_refuses_overlaps(pkg, cuda_dev):
    rec = pkg.recurrence
    i = make_scan([40, 60], 64, torch.bfloat16, cuda_dev)
    want = rec.launch_scan(*gates(i), i["cu"], i["state"])
    buf = torch.zeros(101, 64, dtype=torch.bfloat16, device=cuda_dev)
    buf[:-1] = i["x"]
    j = {**i, "x": buf[:-1]}
    with pytest.raises(ValueError, match="overlap"):
        rec.launch_scan(*gates(j), i["cu"], i["state"], output=buf[1:])
    with pytest.raises(ValueError, match="overlap"):
        rec.launch_scan(*gates(i), i["cu"], i["state"], new_state=want[0].view(-1)[:256].view(torch.float32).view(2, 64), output=want[0])
    wide = torch.zeros(100, 200, dtype=torch.bfloat16, device=cuda_dev)
    with pytest.raises(ValueError, match="overlap"):
        backward(pkg, i, dx=wide[:, :64], da=wide[:, 60:124])
    wide[:, 70:134] = i["x"]
    j = {**i, "x": wide[:, 70:134]}  # between two blocks that are written
    got = rec.launch_scan(*gates(j), i["cu"], i["state"], output=wide[:, 134:198])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    grads = backward(pkg, i)
    got = backward(pkg, j, dx=wide[:, 6:70], da=wide[:, 134:198])
    assert all(torch.equal(a, b) for a, b in zip(got, grads)) and torch.equal(j["x"], i["x"])
    i = make_scan([1] * 6, 64, torch.bfloat16, cuda_dev)
    y, ns = rec.launch_step(*gates(i), i["state"])
    states = torch.zeros(7, 64, device=cuda_dev)
    states[:6] = i["state"]
    with pytest.raises(ValueError, match="overlap"):
        rec.launch_step(*gates(i), states[:6], new_state=states[1:])
    y2, _ = rec.launch_step(*gates(i), states[:6], new_state=states[:6], output=i["x"])
    assert y2 is i["x"] and torch.equal(y2, y) and torch.equal(states[:6], ns)


@gpu
@pytest.mark.parametrize("width", [256, 1003])
def test_norms_refuse_overlaps(pkg, cuda_dev, width):
    n = pkg.norm
    x, res, w = make(40, width, torch.bfloat16, cuda_dev)
    dy = rnd(40, width, dtype=torch.bfloat16, device=cuda_dev, seed=8)
    y, r = n.launch_add_norm(x, res, w, EPS)
    dx, dw = n.launch_add_norm_backward(dy, r, w, EPS, d_new_residual=res)
    buf = torch.zeros(41, width, dtype=torch.bfloat16, device=cuda_dev)
    buf[:-1] = x
    for kw in (dict(output=buf[1:]), dict(new_residual=buf[1:])):
        with pytest.raises(ValueError, match="overlap"):
            n.launch_add_norm(buf[:-1], res, w, EPS, **kw)
    with pytest.raises(ValueError, match="overlap"):
        n.launch_add_norm_backward(dy, buf[:-1], w, EPS, dx=buf[1:])
    wide = torch.zeros(40 * (width + 8), dtype=torch.bfloat16, device=cuda_dev)
    apart = wide.view(40, width + 8)[:, :width]  # begins where `dense` does, rows elsewhere
    dense = wide[:40 * width].view(40, width)
    apart.copy_(x)
    with pytest.raises(ValueError, match="overlap"):
        n.launch_add_norm(apart, res, w, EPS, new_residual=dense)
    assert torch.equal(apart, x)
    # in place, every input in turn
    for k in range(2):
        a, b = x.clone(), res.clone()
        got = n.launch_add_norm(a, b, w, EPS, output=(a, b)[k], new_residual=(b, a)[k])
        assert torch.equal(got[0], y) and torch.equal(got[1], r)
    for k in range(3):
        t = [dy.clone(), r.clone(), res.clone()]
        got = n.launch_add_norm_backward(t[0], t[1], w, EPS, d_new_residual=t[2], dx=t[k])
        assert got[0] is t[k] and torch.equal(got[0], dx) and torch.equal(got[1], dw)


@gpu
def test_gated_norm_refuses_overlaps(pkg, cuda_dev):
    n = pkg.norm
    x, z, dy = (rnd(40, 3, 128, dtype=torch.bfloat16, device=cuda_dev, seed=s) for s in (1, 2, 3))
    w = 1 + rnd(128, device=cuda_dev, scale=0.1)
    grads = n.launch_gated_norm_backward(dy, x, z, w, EPS)
    buf = torch.zeros(41, 3, 128, dtype=torch.bfloat16, device=cuda_dev)
    buf[:-1] = x
    with pytest.raises(ValueError, match="overlap"):
        n.launch_gated_norm(buf[:-1], z, w, EPS, output=buf[1:])
    for kw in (dict(dx=buf[1:]), dict(dz=buf[1:])):
        with pytest.raises(ValueError, match="overlap"):
            n.launch_gated_norm_backward(dy, buf[:-1], z, w, EPS, **kw)
    with pytest.raises(ValueError, match="overlap"):
        n.launch_gated_norm_backward(dy, x, z, w, EPS, dx=buf[1:], dz=buf[:-1])
    for a, b in ((0, 1), (1, 2), (2, 0), (2, 1)):
        t = [dy.clone(), x.clone(), z.clone()]
        got = n.launch_gated_norm_backward(*t, w, EPS, dx=t[a], dz=t[b])
        assert all(torch.equal(g, want) for g, want in zip(got, grads))


@gpu
def test_out_norm_is_refused_before_the_recurrence(pkg, cuda_dev):
    """Whatever the norm cannot take is found while an in-place state is still the state before."""
    w = 1 + rnd(129, device=cuda_dev, scale=0.1)
    dec = pkg.inputs.make_decode_inputs(5, seed=1).to(cuda_dev)
    before = dec.state.clone()
    buf = torch.zeros(6, 8, 128, dtype=torch.bfloat16, device=cuda_dev)
    out, apart = buf[:5], torch.zeros(5, 8, 128, dtype=torch.bfloat16, device=cuda_dev)
    codes = torch.zeros(5, 8, 128, dtype=torch.float8_e4m3fn, device=cuda_dev)
    scale = torch.zeros(5, 8, device=cuda_dev)
    N = pkg.norm.OutputNorm
    for norm in (N(buf[1:], w[:128]), N(buf[1:], w[:128], codes=codes, scale=scale),
                 N(apart, out.view(-1).view(torch.float32)[3:131]), N(apart, w[:128], codes=codes, scale=codes.view(-1)[:160].view(torch.float32).view(5, 8)),
                 N(apart, w[:128], codes=apart.view(torch.float8_e4m3fn).view(-1)[:5120].view(5, 8, 128), scale=scale)):
        with pytest.raises(ValueError, match="overlap|must not be z"):
            pkg.decode.launch_gdn(*dec.args(), output=out, new_state=dec.state, out_norm=norm)
        assert torch.equal(dec.state, before) and not out.any()
    z = rnd(5, 8, 128, dtype=torch.bfloat16, device=cuda_dev)
    pkg.decode.launch_gdn(*dec.args(), output=out, new_state=dec.state, out_norm=N(z, w[1:]))
    assert out.any() and not torch.equal(dec.state, before)


def test_gated_norm_check(pkg):
    """The check answers as the launch does where that refuses, and needs no device where it does not."""
    lib, C = pkg._capi.load(), pkg._capi
    buf = ctypes.create_string_buffer(1 << 14)
    p = (ctypes.addressof(buf) + 4095) // 4096 * 4096
    for want, kw in ((0, {}), (0, dict(output=p)), (0, dict(quant=2)), (0, dict(tokens=0, x=None, z=None, output=None)), (1, dict(z=None)),
                     (1, dict(output=None)), (1, dict(quant=2, scale=None)), (2, dict(head_dim=96)), (2, dict(eps=-1.0)), (3, dict(z=p + 1)),
                     (6, dict(dtype=5)), (8, dict(output=p + 512)), (8, dict(output=p, quant=2)), (8, dict(z=p + 5120, output=p + 5120 + 256))):
        a = C.GdnGatedNormArgs(p, p + 1024, 256, 256, p + 2048, C.DTYPE_F32, C.DTYPE_BF16, 0, EPS, 2, 2, 128, p + 4096, p + 6144)
        for k, v in kw.items():
            setattr(a, k, v)
        assert lib.gdn_gated_norm_check(ctypes.byref(a)) == want, kw
        if want:
            assert lib.gdn_gated_norm_launch(ctypes.byref(a), None) == want, kw
    assert lib.gdn_gated_norm_check(None) == 1
