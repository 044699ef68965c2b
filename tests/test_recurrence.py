"""The per-channel gated recurrence against its definition in 64 bits."""
import bisect
import ctypes

import pytest
import torch

from tests import _layer_ref as ref

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
gpu = pytest.mark.gpu


def make(lens, C, dtype, device="cpu", state=True, seed=0, tail=0, head=0, memory="mixed", fused=False):
    """Inputs of packed sequences; ``head`` and ``tail`` tokens belong to none."""
    gen = torch.Generator().manual_seed(seed)
    T, N = sum(lens) + head + tail, len(lens)
    n = lambda *s, scale=1.0: torch.randn(s, generator=gen) * scale  # noqa: E731
    if fused:
        p = n(T, 3 * C).to(device, dtype)
        x, a, b = p[:, :C], p[:, C:2 * C], p[:, 2 * C:]
    else:
        x, a, b = (n(T, C).to(device, dtype) for _ in range(3))
    A_log = torch.log(torch.rand(C, generator=gen) * 15 + 1)
    lo, hi = {"mixed": (1e-3, 1e-1), "short": (0.5, 4.0)}[memory]
    step = lo * (hi / lo) ** torch.rand(C, generator=gen)
    dt_bias = step + torch.log(-torch.expm1(-step))
    cu = torch.tensor([0] + lens).cumsum(0) + head
    return dict(x=x, A_log=A_log.to(device), a=a, dt_bias=dt_bias.to(device), b=b, lens=lens, first=head,
                cu=cu.to(device), state=n(N, C, scale=0.5).to(device) if state else None,
                dy=n(T, C).to(device, dtype), dns=n(N, C).to(device))


def gates(i):
    return i["x"], i["A_log"], i["a"], i["dt_bias"], i["b"]


def values(i, **kw):
    return ref.scan(*gates(i), i["lens"], i["state"], first=i["first"], **kw)


def check_forward(pkg, i, **kw):
    y, ns = pkg.recurrence.launch_scan(*gates(i), i["cu"], i["state"], **kw)
    want = values(i)
    ref.close(y, *want["y"], "y")
    ref.close(ns, *want["new_state"], "new_state")
    return y, ns


def backward(pkg, i, dns=True, **kw):
    rec = pkg.recurrence
    ck = rec.empty_checkpoints(i["x"])
    rec.launch_scan(*gates(i), i["cu"], i["state"], checkpoints=ck)
    return rec.launch_scan_backward(i["dy"], *gates(i), i["cu"], i["state"], ck, i["dns"] if dns else None, **kw)


def check_backward(pkg, i, dns=True):
    got = backward(pkg, i, dns)
    want = values(i, dy=i["dy"], dns=i["dns"] if dns else None)
    for g, name in zip(got, ("dx", "da", "db", "dA_log", "d_dt_bias", "d_state")):
        if name == "d_state" and i["state"] is None:
            assert g is None
        else:
            ref.close(g, *want[name], name)
    return got


# lengths that meet the edges of the kernels' pieces and tiles (60 and 120 tokens backward, 76 and 152 forward), and
# sequences of nothing
LENS = [[1], [0], [2, 0, 0, 1], [59], [60], [61], [120], [121], [127], [128], [129], [5, 123, 128, 1, 255], [700], [64, 3, 0, 300, 1, 1, 1, 90], [1] * 200,
        [75], [76], [77], [151], [152], [153], [305], [76, 76, 1, 151], [1, 152, 3, 305]]


@gpu
@pytest.mark.parametrize("N", [1022, 1023, 1024, 1025])
def test_scan_of_many_sequences(pkg, cuda_dev, N):
    """Up to 1023 sequences the kernels keep the offsets in shared memory."""
    i = make([(k * 7) % 4 for k in range(N)], 40, torch.bfloat16, cuda_dev)
    check_forward(pkg, i)
    check_backward(pkg, i)


@gpu
@pytest.mark.parametrize("lens", LENS, ids=lambda v: "x".join(map(str, v))[:24])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_scan_forward_and_backward(pkg, cuda_dev, lens, dtype):
    i = make(lens, 72, dtype, cuda_dev)
    check_forward(pkg, i)
    check_backward(pkg, i)


@gpu
@pytest.mark.parametrize("C", [1, 2, 7, 8, 63, 64, 65, 128, 200, 1001])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_scan_channel_counts(pkg, cuda_dev, C, dtype):
    i = make([40, 0, 133, 90], C, dtype, cuda_dev, seed=C)
    check_forward(pkg, i)
    check_backward(pkg, i)


@gpu
@pytest.mark.parametrize("lens", [[9000], [3000, 1, 0, 5200], [2500] * 3], ids=["one", "ragged", "even"])
@pytest.mark.parametrize("C", [64, 130])
def test_scan_long(pkg, cuda_dev, lens, C):
    i = make(lens, C, torch.bfloat16, cuda_dev, seed=3)
    check_forward(pkg, i)
    check_backward(pkg, i)


@gpu
def test_scan_many_short_sequences(pkg, cuda_dev):
    """More sequences than a block could hold offsets for."""
    lens = [k % 4 for k in range(5000)]
    i = make(lens, 66, torch.bfloat16, cuda_dev, seed=4)
    check_forward(pkg, i)
    check_backward(pkg, i)


@gpu
@pytest.mark.parametrize("state", [True, False])
@pytest.mark.parametrize("dns", [True, False])
def test_scan_without_states(pkg, cuda_dev, state, dns):
    i = make([30, 200], 64, torch.bfloat16, cuda_dev, state=state)
    check_forward(pkg, i)
    check_backward(pkg, i, dns)


@gpu
@pytest.mark.parametrize("cu_dtype", [torch.int32, torch.int64])
def test_scan_seqlens_types_and_cpu_seqlens(pkg, cuda_dev, cu_dtype):
    i = make([30, 200], 64, torch.bfloat16, cuda_dev)
    want = check_forward(pkg, i)
    i["cu"] = i["cu"].to(cu_dtype)
    for cu in (i["cu"], i["cu"].cpu()):
        i["cu"] = cu
        got = check_forward(pkg, i)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@gpu
@pytest.mark.parametrize("head,tail", [(0, 5), (3, 0), (130, 260), (0, 1000)])
def test_scan_tokens_of_no_sequence(pkg, cuda_dev, head, tail):
    """Their rows and gradients are zeros, whatever they hold, and they reach nobody."""
    i = make([30, 0, 150], 64, torch.bfloat16, cuda_dev, head=head, tail=tail)
    for k in ("x", "a", "b", "dy"):
        i[k][:head] = float("nan")
        i[k][head + 180:] = float("inf")
    out = torch.full_like(i["x"], 7.0)
    y, ns = pkg.recurrence.launch_scan(*gates(i), i["cu"], i["state"], output=out)
    clean = make([30, 0, 150], 64, torch.bfloat16, cuda_dev, head=head, tail=tail)
    want = values(clean)
    sl = slice(head, head + 180)
    ref.close(y[sl], want["y"][0][sl], want["y"][1][sl], "y")
    ref.close(ns, *want["new_state"], "new_state")
    assert not y[:head].any() and not y[head + 180:].any()
    got = backward(pkg, i)
    wantg = values(clean, dy=clean["dy"], dns=clean["dns"])
    for g, name in zip(got, ("dx", "da", "db")):
        assert not g[:head].any() and not g[head + 180:].any(), name
        ref.close(g[sl], wantg[name][0][sl], wantg[name][1][sl], name)
    for g, name in zip(got[3:], ("dA_log", "d_dt_bias", "d_state")):
        assert bool(g.isfinite().all()), name


@gpu
@pytest.mark.parametrize("lens", [[40, 100, 3, 200], [40, 130, 20, 300], [3, 250, 9, 9, 9, 300], [1, 125, 8, 8, 8, 8, 400]],
                         ids=lambda v: "x".join(map(str, v)))
@pytest.mark.parametrize("C", [64, 1024])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
def test_scan_sequences_do_not_leak(pkg, cuda_dev, lens, C, dtype):
    """NaN and infinity in the second sequence leave its neighbours alone, forward and backward, with any
    number of sequences starting in the tile where it ends."""
    i = make(lens, C, dtype, cuda_dev)
    T, N, t0, t1 = sum(lens), len(lens), lens[0], lens[0] + lens[1]
    others = [n for n in range(N) if n != 1]
    good = pkg.recurrence.launch_scan(*gates(i), i["cu"], i["state"])
    good_grads = backward(pkg, i)
    keep = torch.ones(T, dtype=torch.bool, device=cuda_dev)
    keep[t0:t1] = False
    for bad in (float("nan"), float("inf")):
        j = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in i.items()}
        j["x"][t0 + 20] = bad
        j["state"][1] = bad
        j["dy"][t0 + 30] = bad
        j["dns"][1] = bad
        y, ns = pkg.recurrence.launch_scan(*gates(j), j["cu"], j["state"])
        assert torch.equal(y[keep], good[0][keep]) and not y[t0 + 20].isfinite().any()
        assert torch.equal(ns[others], good[1][others])
        grads = backward(pkg, j)
        for g, w in zip(grads[:3], good_grads[:3]):
            assert torch.equal(g[keep], w[keep])
        assert torch.equal(grads[5][others], good_grads[5][others])


@gpu
def test_scan_extreme_gates(pkg, cuda_dev):
    """Gates that open or close entirely; infinite pre-activations are limits."""
    i = make([300], 64, torch.float32, cuda_dev, memory="short")
    i["a"][10:20] = 300.0     # g = 0
    i["a"][50:60] = -300.0    # g = 1
    i["a"][100] = float("inf")
    i["a"][101] = -float("inf")
    i["b"][30:40] = 200.0
    i["b"][70:80] = -200.0
    i["b"][110] = float("inf")
    i["b"][111] = -float("inf")
    y, ns = pkg.recurrence.launch_scan(*gates(i), i["cu"], i["state"])
    fin = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in i.items()}
    for k in ("a", "b"):
        fin[k] = fin[k].clamp(-1e4, 1e4)
    want = values(fin)
    ref.close(y, *want["y"], "y")
    ref.close(ns, *want["new_state"], "new_state")


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("C", [64, 72, 65])
def test_scan_strided_inputs_and_outputs(pkg, cuda_dev, dtype, C):
    """Column blocks of one projection in, column blocks of a wider buffer out; nothing beside them is touched."""
    i = make([40, 133], C, dtype, cuda_dev, fused=True)
    wide = torch.full((173, C + 24), 7.0, dtype=dtype, device=cuda_dev)
    check_forward(pkg, i, output=wide[:, 16:16 + C])
    assert bool((wide[:, :16] == 7).all()) and bool((wide[:, 16 + C:] == 7).all())
    g = torch.full((173, 3 * C + 1), 7.0, dtype=dtype, device=cuda_dev)
    got = backward(pkg, i, dx=g[:, :C], da=g[:, C:2 * C], db=g[:, 2 * C:3 * C])
    dense = backward(pkg, i)
    for a, b in zip(got, dense):
        assert torch.equal(a, b)
    assert bool((g[:, 3 * C:] == 7).all())


@gpu
def test_scan_unaligned_base(pkg, cuda_dev):
    i = make([40, 133], 64, torch.bfloat16, cuda_dev)
    want = pkg.recurrence.launch_scan(*gates(i), i["cu"], i["state"])
    for k in ("x", "a", "b"):
        buf = torch.empty(173 * 64 + 3, dtype=torch.bfloat16, device=cuda_dev)
        buf[3:] = i[k].flatten()
        i[k] = buf[3:].view(173, 64)
    got = pkg.recurrence.launch_scan(*gates(i), i["cu"], i["state"])
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@gpu
def test_scan_offsets_past_32_bits(pkg, cuda_dev):
    C, T, wide = 64, 40000, 65536
    big = torch.empty((T, wide), dtype=torch.bfloat16, device=cuda_dev)  # 2.6e9 elements
    i = make([T - 100, 100], C, torch.bfloat16, cuda_dev)
    want = pkg.recurrence.launch_scan(*gates(i), i["cu"], i["state"])
    big[:, -C:] = i["x"]
    i["x"] = big[:, -C:]
    got = pkg.recurrence.launch_scan(*gates(i), i["cu"], i["state"])
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@gpu
def test_scan_chains_like_one_call(pkg, cuda_dev):
    """A prefix, its state, the rest, then steps: the values of the whole sequence."""
    i = make([400], 64, torch.float32, cuda_dev)
    rec, want = pkg.recurrence, values(i)
    x, A, a, d, b = gates(i)
    cu = lambda n: torch.tensor([0, n], device=cuda_dev)  # noqa: E731
    y0, s = rec.launch_scan(x[:150], A, a[:150], d, b[:150], cu(150), i["state"])
    y1, s = rec.launch_scan(x[150:390], A, a[150:390], d, b[150:390], cu(240), s)
    ys = []
    for t in range(390, 397):
        y, s = rec.launch_step(x[t:t + 1], A, a[t:t + 1], d, b[t:t + 1], s, new_state=s)
        ys.append(y)
    y3, s = rec.launch_step(x[None, 397:], A, a[None, 397:], d, b[None, 397:], s)
    y = torch.cat([y0, y1, *ys, y3[0]])
    # a split adds one association; the bound leaves a factor of two for that
    ref.close(y, *want["y"], "y")
    ref.close(s, *want["new_state"], "new_state")


@gpu
@pytest.mark.parametrize("B", [1, 3, 256])
@pytest.mark.parametrize("C", [1, 65, 128, 1000, 4096])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_step(pkg, cuda_dev, B, C, dtype):
    i = make([1] * B, C, dtype, cuda_dev, seed=B)
    want = values(i)
    y, ns = pkg.recurrence.launch_step(*gates(i), i["state"])
    ref.close(y, *want["y"], "y")
    ref.close(ns, *want["new_state"], "new_state")
    inplace = i["state"].clone()
    y2, ns2 = pkg.recurrence.launch_step(*gates(i), inplace, new_state=inplace)
    assert ns2 is inplace and torch.equal(inplace, ns) and torch.equal(y2, y)


@gpu
def test_step_tokens_and_strides(pkg, cuda_dev):
    i = make([5] * 7, 96, torch.bfloat16, cuda_dev, fused=True)
    want = values(i)
    x, A, a, d, b = gates(i)
    v = lambda t: t.unflatten(0, (7, 5))  # noqa: E731
    y, ns = pkg.recurrence.launch_step(v(x), A, v(a), d, v(b), i["state"])
    assert y.shape == (7, 5, 96)
    ref.close(y.flatten(0, 1), *want["y"], "y")
    ref.close(ns, *want["new_state"], "new_state")


@gpu
def test_empty_calls(pkg, cuda_dev):
    rec = pkg.recurrence
    z = torch.zeros(0, 64, dtype=torch.bfloat16, device=cuda_dev)
    v = torch.zeros(64, device=cuda_dev)
    s = torch.randn(3, 64, device=cuda_dev)
    cu = torch.zeros(4, dtype=torch.int64, device=cuda_dev)
    y, ns = rec.launch_scan(z, v, z, v, z, cu, s)
    assert y.shape == (0, 64) and torch.equal(ns, s)
    assert not rec.launch_scan(z, v, z, v, z, cu)[1].any()
    g = rec.launch_scan_backward(z, z, v, z, v, z, cu, s, rec.empty_checkpoints(z), d_new_state=s)
    assert torch.equal(g[5], s) and not g[3].any() and not g[4].any()
    x = torch.ones(5, 64, dtype=torch.bfloat16, device=cuda_dev)
    y, ns = rec.launch_scan(x, v, x, v, x, cu[:1])
    assert not y.any() and ns.shape == (0, 64)
    g = rec.launch_scan_backward(x, x, v, x, v, x, cu[:1], None, rec.empty_checkpoints(x))
    assert not any(t.any() for t in g[:5])
    y, ns = rec.launch_step(z, v, z, v, z, torch.zeros(0, 64, device=cuda_dev))
    assert y.shape == (0, 64)


@gpu
def test_scan_is_reproducible_and_uses_the_current_stream(pkg, cuda_dev):
    i = make([3000, 17, 2000], 256, torch.bfloat16, cuda_dev)
    y0, n0 = pkg.recurrence.launch_scan(*gates(i), i["cu"], i["state"])
    g0 = backward(pkg, i)
    side = torch.cuda.Stream(cuda_dev)
    side.wait_stream(torch.cuda.current_stream(cuda_dev))
    with torch.cuda.stream(side):
        torch.cuda._sleep(2_000_000)
        j = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in i.items()}
        for _ in range(4):
            y, n = pkg.recurrence.launch_scan(*gates(j), j["cu"], j["state"])
            g = backward(pkg, j)
    side.synchronize()
    assert torch.equal(y, y0) and torch.equal(n, n0)
    for a, b in zip(g, g0):
        assert torch.equal(a, b)


@gpu
def test_two_calls_at_once(pkg, cuda_dev):
    i, j = (make([2000, 900], 512, torch.bfloat16, cuda_dev, seed=s) for s in (1, 2))
    want = [backward(pkg, k) for k in (i, j)]
    streams = [torch.cuda.Stream(cuda_dev) for _ in range(2)]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(3):
        for k, (s, inp) in enumerate(zip(streams, (i, j))):
            with torch.cuda.stream(s):
                got[k] = backward(pkg, inp)
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        for a, b in zip(g, w):
            assert torch.equal(a, b)


@gpu
def test_scan_in_two_graphs(pkg, cuda_dev):
    """Two captured training passes with buffers of their own, replayed in turn on new data."""
    rec = pkg.recurrence
    pair = [make([300, 50], 64, torch.bfloat16, cuda_dev, seed=s) for s in (1, 2)]
    outs, graphs = [], []
    for i in pair:
        backward(pkg, i)  # warm up
    torch.cuda.synchronize()
    for i in pair:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append((rec.launch_scan(*gates(i), i["cu"], i["state"]), backward(pkg, i)))
        graphs.append(g)
    for i in pair:
        i["x"].neg_()
        i["dy"].mul_(2)
    for _ in range(2):
        for g in graphs:
            g.replay()
    torch.cuda.synchronize()
    for i, ((y, ns), grads) in zip(pair, outs):
        want = values(i, dy=i["dy"], dns=i["dns"])
        ref.close(y, *want["y"], "y")
        ref.close(ns, *want["new_state"], "new_state")
        for g, name in zip(grads, ("dx", "da", "db", "dA_log", "d_dt_bias", "d_state")):
            ref.close(g, *want[name], name)


@gpu
def test_gated_scan_gradients(pkg, cuda_dev):
    """The differentiable form gives the launch functions' gradients, and those follow differences."""
    i = make([20, 150], 8, torch.float32, cuda_dev, memory="short")
    leaves = [i[k].clone().requires_grad_() for k in ("x", "A_log", "a", "dt_bias", "b")]
    s = i["state"].clone().requires_grad_()
    y, ns = pkg.recurrence.gated_scan(*leaves, i["cu"], s)
    ((y * i["dy"]).sum() + (ns * i["dns"]).sum()).backward()
    dx, da, db, dA, ddt, ds = backward(pkg, i)
    for leaf, want in zip(leaves + [s], (dx, dA, da, ddt, db, ds)):
        assert torch.equal(leaf.grad, want)

    def loss(**kw):
        j = {**i, **kw}
        w = ref.scan(*gates(j), j["lens"], j["state"])
        return float((w["y"][0] * i["dy"].double()).sum() + (w["new_state"][0] * i["dns"].double()).sum())

    gen = torch.Generator().manual_seed(5)
    for name, grad in (("x", dx), ("a", da), ("b", db), ("A_log", dA), ("dt_bias", ddt), ("state", ds)):
        v = torch.randn(grad.shape, generator=gen, dtype=torch.float64).to(cuda_dev)
        h = 1e-5  # central differences of a 64-bit loss: h^2 of the third derivative, 1e-16 / h of rounding
        slope = (loss(**{name: i[name].double() + h * v}) - loss(**{name: i[name].double() - h * v})) / (2 * h)
        scale = float(grad.double().norm() * v.norm()) / grad.numel() ** 0.5
        assert abs(slope - float((grad.double() * v).sum())) <= 1e-4 * scale, name


@gpu
def test_gated_scan_partial_gradients(pkg, cuda_dev):
    """Only the state's output is used; an expanded gradient; no state."""
    i = make([20, 150], 64, torch.bfloat16, cuda_dev, state=False)
    x = i["x"].clone().requires_grad_()
    y, ns = pkg.recurrence.gated_scan(x, *gates(i)[1:], i["cu"])
    ns.sum().backward()
    j = {**i, "dy": torch.zeros_like(i["dy"]), "dns": torch.ones_like(i["dns"])}
    assert torch.equal(x.grad, backward(pkg, j)[0])
    x.grad = None
    y, ns = pkg.recurrence.gated_scan(x, *gates(i)[1:], i["cu"])
    y.float().sum().backward()
    j = {**i, "dy": torch.ones_like(i["dy"])}
    assert torch.equal(x.grad, backward(pkg, j, dns=False)[0])


@gpu
@pytest.mark.parametrize("cu", [[0, 50, 40], [-5, 50, 90], [0, 50, 91], [0, 1000, 90]], ids=str)
def test_bad_seqlens_are_reported(pkg, cuda_dev, cu):
    i = make([50, 40], 64, torch.bfloat16, cuda_dev)
    i["cu"] = torch.tensor(cu, device=cuda_dev)
    assert pkg.prefill.device_status(cuda_dev) == 0
    pkg.recurrence.launch_scan(*gates(i), i["cu"], i["state"])
    assert pkg.prefill.device_status(cuda_dev) == pkg._capi.GDN_ERR_DEVICE_BAD_SEQLENS
    backward(pkg, i)
    assert pkg.prefill.device_status(cuda_dev) == pkg._capi.GDN_ERR_DEVICE_BAD_SEQLENS
    with pytest.raises(ValueError, match="cu_seqlens"):
        pkg.recurrence.launch_scan(*gates(i), i["cu"], i["state"], check_seqlens=True)
    i["cu"] = torch.tensor([0, 50, 90], device=cuda_dev)
    check_forward(pkg, i)
    assert pkg.prefill.device_status(cuda_dev) == 0


# ---------------------------------------------------------------- refusals --
def _refuse(pkg, match, i, **kw):
    args = dict(output=torch.empty_like(i["x"]), new_state=torch.empty(2, 16), require_cuda=False)
    args.update(kw)
    with pytest.raises(ValueError, match=match):
        pkg.recurrence.validate(*gates(i), i["cu"], i["state"], **args)


def test_scan_refusals(pkg):
    i = make([4, 6], 16, torch.bfloat16)
    ok = dict(output=torch.empty_like(i["x"]), new_state=torch.empty(2, 16), require_cuda=False)
    assert pkg.recurrence.validate(*gates(i), i["cu"], i["state"], **ok, check_seqlens=True) == (10, 2, 16)
    with pytest.raises(ValueError, match="CUDA tensor"):
        pkg.recurrence.launch_scan(*gates(i), i["cu"], i["state"])
    with pytest.raises(ValueError, match="CUDA tensor"):
        pkg.recurrence.launch_step(*gates(i), i["state"])
    _refuse(pkg, "x must be a", {**i, "x": i["x"][0]})
    _refuse(pkg, "bfloat16, float16 or float32", {**i, "x": i["x"].double()})
    _refuse(pkg, "a must be torch.bfloat16", {**i, "a": i["a"].float()})
    _refuse(pkg, "b must have shape", {**i, "b": i["b"][:5]})
    _refuse(pkg, "contiguous rows", {**i, "a": i["a"].t().contiguous().t()})
    _refuse(pkg, "overlapping rows", {**i, "a": i["a"][:1].expand(10, 16)})
    _refuse(pkg, "A_log must be torch.float32", {**i, "A_log": i["A_log"].double()})
    _refuse(pkg, "dt_bias must have shape", {**i, "dt_bias": i["dt_bias"][:3]})
    _refuse(pkg, "int32 or int64", {**i, "cu": i["cu"].float()})
    _refuse(pkg, "N\\+1 offsets", {**i, "cu": i["cu"][:0]})
    _refuse(pkg, "state must have shape", {**i, "state": i["state"][:1]})
    _refuse(pkg, "state must be torch.float32", {**i, "state": i["state"].bfloat16()})
    _refuse(pkg, "must not alias", i, new_state=i["state"])
    _refuse(pkg, "must not overlap", i, output=i["x"])
    _refuse(pkg, "checkpoints must have shape", i, checkpoints=torch.empty(3, 16))
    _refuse(pkg, "exceeds total tokens", {**i, "cu": torch.tensor([0, 4, 11])}, check_seqlens=True)
    _refuse(pkg, "non-decreasing", {**i, "cu": torch.tensor([0, 6, 4])}, check_seqlens=True)


@gpu
@pytest.mark.parametrize("same", [("dx", "da"), ("da", "db"), ("dx", "db")])
def test_scan_gradients_apart(pkg, cuda_dev, same):
    i = make([4, 6], 16, torch.bfloat16, cuda_dev)
    out = torch.empty_like(i["x"])
    with pytest.raises(ValueError, match="another gradient"):
        backward(pkg, i, **dict.fromkeys(same, out))
    with pytest.raises(ValueError, match="must not overlap an input"):
        backward(pkg, i, **{same[0]: i["dy"]})


def test_scan_capi_refusals(pkg):
    """Host-side checks come before any device call, so they answer without a GPU."""
    lib, C = pkg._capi.load(), pkg._capi
    buf = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(buf) + 63) // 64 * 64

    def args(**kw):
        a = C.GdnScanArgs(p, p, p, 16, 16, 16, p, p, None, p, C.GDN_SEQLENS_INT64, C.DTYPE_BF16, 4, 2, 16, p, 16, p + 256, p)
        for k, v in kw.items():
            setattr(a, k, v)
        return ctypes.byref(a)

    def grads(**kw):
        g = C.GdnScanGradArgs(p, 16, None, p, p, p, 16, 16, 16, p, p, None)
        for k, v in kw.items():
            setattr(g, k, v)
        return ctypes.byref(g)

    NULL, SIZE, ALIGN, DTYPE = 1, 2, 3, 6
    for want, kw in [(NULL, dict(x=None)), (NULL, dict(A_log=None)), (NULL, dict(cu_seqlens=None)), (NULL, dict(output=None)),
                     (NULL, dict(new_state=None)), (SIZE, dict(total_tokens=-1)), (SIZE, dict(num_seqs=-1)),
                     (SIZE, dict(channels=0)), (SIZE, dict(channels=1 << 21)), (SIZE, dict(x_stride=15)),
                     (SIZE, dict(output_stride=15)), (SIZE, dict(state=p + 256)), (ALIGN, dict(x=p + 1)),
                     (ALIGN, dict(cu_seqlens=p + 4)), (ALIGN, dict(new_state=p + 2)), (DTYPE, dict(dtype=3)),
                     (DTYPE, dict(cu_seqlens_dtype=2))]:
        assert lib.gdn_scan_launch(args(**kw), None) == want, kw
    assert lib.gdn_scan_launch(None, None) == NULL
    for want, kw in [(NULL, dict(dx=None)), (NULL, dict(d_output=None)), (NULL, dict(dA_log=None)), (SIZE, dict(da_stride=3)),
                     (ALIGN, dict(db=p + 1)), (ALIGN, dict(d_state=p + 2))]:
        assert lib.gdn_scan_backward_launch(args(), grads(**kw), None) == want, kw
    assert lib.gdn_scan_backward_launch(args(), None, None) == NULL
    assert lib.gdn_scan_backward_launch(args(checkpoints=None), grads(), None) == NULL
    step = dict(total_tokens=2, state=p)
    assert lib.gdn_scan_step_launch(args(**step), 0, None) == SIZE
    assert lib.gdn_scan_step_launch(args(**step), 2, None) == SIZE
    assert lib.gdn_scan_step_launch(args(**{**step, "state": None}), 1, None) == NULL
    assert lib.gdn_scan_checkpoint_rows(0) == 0 and lib.gdn_scan_checkpoint_rows(129) == 3


def test_bounds_follow_fp32(pkg):
    """The oracle's bounds hold for a plain fp32 evaluation, and notice a wrong gate."""
    i = make([60, 0, 41], 12, torch.float32)
    want = values(i, dy=i["dy"], dns=i["dns"])
    x, A_log, a, dt, b = gates(i)
    sp = torch.nn.functional.softplus(a + dt, threshold=1000.0)
    g, beta = torch.exp(-A_log.exp() * sp), torch.sigmoid(b)
    h, ys = i["state"].clone(), []
    for n, (t0, t1) in enumerate(((0, 60), (60, 60), (60, 101))):
        for t in range(t0, t1):
            h[n] = g[t] * h[n] + beta[t] * x[t]
            ys.append(h[n].clone())
    y = torch.stack(ys)
    ref.close(y, *want["y"], "y")
    ref.close(h, *want["new_state"], "new_state")
    with pytest.raises(AssertionError):
        ref.close(y * (1 + 1e-4), *want["y"], "y")


# --------------------------------------------------------- leaving a cluster --
def _kernel_bodies(source):
    """Bodies of the __global__ functions that use distributed shared memory, by name."""
    out, at = {}, 0
    while (at := source.find("__global__", at)) >= 0:
        open_ = source.index("{", at)
        depth, end = 1, open_ + 1
        while depth:
            depth += {"{": 1, "}": -1}.get(source[end], 0)
            end += 1
        body = source[open_ + 1:end - 1]
        if "st_cluster_f4" in body:
            out[source[at:open_].split("(")[-2].split()[-1]] = body
        at = end
    return out


def test_scans_leave_their_cluster_together(pkg):
    """A wait that runs out is not forced on a GPU; that its CTA stays for its peers is held here.  No thread of a scan
    ends but behind the cluster's barrier, the kernel's last statement, and every wait answers for its whole warp."""
    source = (pkg._build.CSRC / "gdn_recurrence.cu").read_text()
    bodies = _kernel_bodies(source)
    assert set(bodies) == {"gdn_scan_kernel", "gdn_scan_backward_kernel"}
    for name, body in bodies.items():
        assert body.rstrip().endswith("leave_cluster(gave_up);") and body.count("leave_cluster") == 1, name
        assert "return;" not in body and "return record_status" not in body, name
        assert "mbar_wait" not in body and body.count("warp_wait(") == body.count("gave_up = !warp_wait(") + body.count("if (warp_wait("), name
    leave = source[source.index("void leave_cluster"):]
    leave = leave[:leave.index("\n}\n")]
    assert leave.index("cluster_arrive") < leave.index("cluster_wait") < leave.index("record_status")


# ---------------------------------------------- many empty sequences in a row --
def _walk(ends, t, width, tokens):
    """The warp's walk over the sequences of one piece (find_spans), in its order: starts, ends, covered, steps."""
    starts, seqs, stop = [0] + ends[:-1], len(ends), min(t + width, tokens)
    start = end = covered = steps = 0
    n = bisect.bisect_right(ends, t)
    while n < seqs:
        steps += 1
        for k in range(n, min(n + 32, seqs)):
            b, e = starts[k], ends[k]
            if e > b and b < stop and e > t:
                start |= (b >= t) << max(b - t, 0)
                end |= (e <= stop) << max(min(e, stop) - 1 - t, 0)
                for j in range(max(b, t), min(e, stop)):
                    covered |= 1 << (j - t)
        last = starts[n + 31] if n + 31 < seqs else stop
        if last >= stop:
            break
        n = max(n + 32, bisect.bisect_right(ends, last))
    return start, end, covered, steps


@pytest.mark.parametrize("width", [4, 8, 16])
def test_walk_over_empty_sequences(pkg, width):
    """The walk's steps are bounded by the piece's tokens, not by the sequences; nothing is missed."""
    gen = torch.Generator().manual_seed(0)
    for case in range(40):
        lens = torch.randint(0, 3 + case % 5, (60,), generator=gen).tolist()
        for k in torch.randint(0, 60, (4,), generator=gen).tolist():
            lens[k:k] = [0] * int(torch.randint(0, 3000, (1,), generator=gen))
        ends = torch.tensor(lens).cumsum(0).tolist()
        tokens = ends[-1] + case % 3
        first = {b for b, n in zip([0] + ends[:-1], lens) if n}
        last = {e - 1 for e, n in zip(ends, lens) if n}
        for t in range(0, tokens, width):
            start, end, covered, steps = _walk(ends, t, width, tokens)
            live = range(min(width, tokens - t))
            assert start == sum(1 << j for j in live if t + j in first)
            assert end == sum(1 << j for j in live if t + j in last)
            assert covered == sum(1 << j for j in live if t + j < ends[-1])
            assert steps <= width + 1


@gpu
@pytest.mark.parametrize("N", [900, 400_000])
def test_scan_of_many_empty_sequences(pkg, cuda_dev, N):
    """Offsets that repeat in the middle of a tile, with and without tokens of other sequences beside them: the bits of
    the call without them, and their state rows passed on."""
    C, gen = 24, torch.Generator().manual_seed(1)
    i = make([101, 3, 1, 140], C, torch.bfloat16, cuda_dev)
    at = [1, N // 3, N // 2 + 40, N + 3]  # where the four stand among the empty ones
    lens = torch.zeros(N + 4, dtype=torch.int64)
    lens[at] = torch.tensor(i["lens"])
    state, dns = (torch.randn(N + 4, C, generator=gen).to(cuda_dev) for _ in range(2))
    state[at], dns[at] = i["state"], i["dns"]
    j = {**i, "cu": torch.cat([torch.zeros(1, dtype=torch.int64), lens.cumsum(0)]).to(cuda_dev), "state": state, "dns": dns}
    for a, b in zip(check_forward(pkg, i), pkg.recurrence.launch_scan(*gates(j), j["cu"], j["state"])):
        assert torch.equal(a, b if a.shape == b.shape else b[at])
    ns = pkg.recurrence.launch_scan(*gates(j), j["cu"], j["state"])[1]
    empty = torch.ones(N + 4, dtype=torch.bool, device=cuda_dev)
    empty[at] = False
    assert torch.equal(ns[empty], state[empty])
    want, got = backward(pkg, i), backward(pkg, j)
    for a, b in zip(want[:5], got[:5]):
        assert torch.equal(a, b)
    assert torch.equal(got[5][at], want[5]) and torch.equal(got[5][empty], dns[empty])
    assert pkg.prefill.device_status(cuda_dev) == 0


# ------------------------------------------------------------------- limits --
def test_scan_refuses_what_its_indices_cannot_hold(pkg):
    """As ``ValueError``, from ``validate`` and from the entry points alike."""
    rec = pkg.recurrence
    i = make([2], 4, torch.bfloat16)
    far = torch.empty_strided((2, 4), (rec.MAX_STRIDE + 2, 1), dtype=torch.bfloat16)  # address space only
    ok = dict(output=torch.empty_like(i["x"]), new_state=torch.empty(1, 4), require_cuda=False)
    for k in ("x", "a", "b"):
        with pytest.raises(ValueError, match=f"{k} must have at most"):
            rec.validate(*gates({**i, k: far}), i["cu"], i["state"], **ok)
    with pytest.raises(ValueError, match="output must have at most"):
        rec.validate(*gates(i), i["cu"], i["state"], **{**ok, "output": far})
    many = rec.MAX_CHANNELS + 1
    x, v = torch.zeros(1, many), torch.zeros(many)
    with pytest.raises(ValueError, match="channels"):
        rec.validate(x, v, x, v, x, torch.tensor([0, 1]), None, torch.empty_like(x), torch.empty(1, many), require_cuda=False)
    for x in (i["x"][0], i["x"][None], None):
        with pytest.raises(ValueError, match="x must be a"):
            rec.empty_checkpoints(x)
        with pytest.raises(ValueError, match="x must be a"):
            rec.gated_scan(x, *gates(i)[1:], i["cu"])


def test_argument_statuses_are_value_errors(pkg):
    C = pkg._capi
    for status in range(1, 64):
        with pytest.raises(C.GdnError) as e:
            C.check(status, "call")
        assert isinstance(e.value, ValueError) == (status in (1, 2, 3, 4, 6, 8)) and e.value.status == status


# ------------------------------------------------- gates far from the middle --
@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("special", [False, True], ids=["inside", "starts"])
def test_db_of_open_gates(pkg, cuda_dev, dtype, special):
    """db = G x sigmoid(b) sigmoid(-b) for b from -60 to 60, where 1 - sigmoid(b) cannot be had by a difference.  Decays
    of zero, so every token's gradient is its own, in pieces inside a sequence and in pieces where some start."""
    T, C = 240, 32
    i = make([1, 2, 3] * 40 if special else [T], C, dtype, cuda_dev, state=False)
    i["b"] = torch.linspace(-60, 60, T * C, device=cuda_dev).view(T, C).to(dtype)
    i["a"] += 300.0
    x, dy, b = (i[k].double() for k in ("x", "dy", "b"))
    beta, rest = torch.sigmoid(b), torch.sigmoid(-b)
    dx, _, db = backward(pkg, i, dns=False)[:3]
    # e = exp(-|b|): 2 U of the exponential and |b| U of its rounded argument; 1 / (1 + e): 2 U; 1 - e / (1 + e) adds U, and
    # its argument's error times e, under U; three products
    err = (12 + b.abs()) * ref.U
    ref.close(dx, dy * beta, err * (dy * beta).abs(), "dx")
    ref.close(db, dy * x * beta * rest, 2 * err * (dy * x * beta * rest).abs(), "db")


@gpu
def test_gates_past_the_exponents(pkg, cuda_dev):
    """b and a at infinities and far out: gradients are the limits, and a NaN stays a NaN in its own channel."""
    T, C = 150, 64
    i = make([T], C, torch.float32, cuda_dev, memory="short", state=False)
    for t, v in ((3, 100.0), (4, -100.0), (70, 1e4), (71, -1e4), (90, float("inf")), (91, -float("inf"))):
        i["b"][t] = v
    got = backward(pkg, i, dns=False)
    fin = {**i, "b": i["b"].clamp(-500, 500)}
    want = values(fin, dy=i["dy"], dns=None)
    for g, name in zip(got, ("dx", "da", "db", "dA_log", "d_dt_bias")):
        ref.close(g, *((v + (2.0 ** -126) * 16 if k else v) for k, v in enumerate(want[name])), name)  # flushed below 2^-126
    j = {**i, "b": i["b"].clone()}
    j["b"][40, 5] = float("nan")
    bad = backward(pkg, j, dns=False)
    keep = torch.arange(C, device=cuda_dev) != 5
    for g, w in zip(bad[:3], got[:3]):
        assert torch.equal(g[:, keep], w[:, keep])
    assert bool(bad[2][40, 5].isnan())


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("C", [64, 1024])
@pytest.mark.parametrize("T", [5, 300, 3000])
def test_infinite_states_stay(pkg, cuda_dev, T, C, dtype):
    """An infinity, of the state before or of a token, is the state until the sequence ends, however small the product
    of its decays; what follows is as without it."""
    inf = float("inf")
    i = make([T, 40, T], C, dtype, cuda_dev, memory="short")
    good = pkg.recurrence.launch_scan(*gates(i), i["cu"], i["state"])
    i["state"][0, :8], i["state"][0, 8:16] = inf, -inf
    at = T + 40 + T // 2
    i["x"][at, 16:24], i["x"][at, 24:32] = inf, -inf
    y, ns = pkg.recurrence.launch_scan(*gates(i), i["cu"], i["state"])
    want, want_ns = good[0].clone(), good[1].clone()
    want[:T, :8], want[:T, 8:16], want_ns[0, :8], want_ns[0, 8:16] = inf, -inf, inf, -inf
    want[at:, 16:24], want[at:, 24:32], want_ns[2, 16:24], want_ns[2, 24:32] = inf, -inf, inf, -inf
    # infinities of two signs meet in a NaN
    assert torch.equal(y, want) and torch.equal(ns, want_ns)
    i["x"][T - 1, :8] = -inf
    y, ns = pkg.recurrence.launch_scan(*gates(i), i["cu"], i["state"])
    assert bool(y[T - 1, :8].isnan().all()) and torch.equal(y[T:], want[T:]) and torch.equal(ns[1:], want_ns[1:])


# ----------------------------------------------- sums with one term to them --
@gpu
@pytest.mark.parametrize("lens", [[1000], [299, 1, 0, 700], [1] * 200], ids=["one", "ragged", "single"])
@pytest.mark.parametrize("C", [40, 1024])
def test_parameter_gradients_of_one_token(pkg, cuda_dev, lens, C):
    """A gradient that enters at one token: the parameters' are then sums of the few terms before it, and a term that
    is lost or counted twice, at a piece's or a tile's edge or at an end, is most of the answer."""
    i = make(lens, C, torch.bfloat16, cuda_dev, memory="short")
    T, U = sum(lens), ref.U
    z = i["a"].double() + i["dt_bias"].double()
    sp, sig = torch.logaddexp(z, torch.zeros_like(z)), torch.sigmoid(z)
    dy = i["dy"]
    # an exponential below 2^-126 is flushed to zero (a = 4.7 at rate 16: g = 2e-42), so a decay is off by that at most, and
    # each of the T terms G g h rate sigmoid(z) by that times |G| |h| rate, |G| <= |dy|
    h = max(float(v.abs().max()) for v in (i["state"], values(i)["y"][0]))
    flush = 2.0 ** -126 * T * float(dy.abs().max()) * h * i["A_log"].double().exp()
    for t in sorted({0, 1, 3, 4, 7, 8, 59, 60, 61, 119, 120, 151, 152, T - 121, T - 61, T - 60, T - 2, T - 1}):
        i["dy"] = torch.zeros_like(dy)
        i["dy"][t] = dy[t]
        got = backward(pkg, i, dns=False)
        da, err = values(i, dy=i["dy"], dns=None)["da"]
        # a thread adds 4 tokens of each of its tiles (9 at most here), then 2 strips, 15 warps, 16 blocks: 71 roundings
        depth = 100 * U
        ref.close(got[4], da.sum(0), err.sum(0) + depth * da.abs().sum(0) + flush, f"d_dt_bias of token {t}")
        # dA_log = sum of dl l = sum of da softplus / sigmoid; l has 8 U and its argument's rounding, sigmoid 8 U
        dA, more = da * sp / sig, (32 + z.abs() * sig / sp) * U
        ref.close(got[3], dA.sum(0), (err * sp / sig + (depth + more) * dA.abs()).sum(0) + flush * sp.amax(0), f"dA_log of token {t}")


def test_gate_polynomials(pkg):
    """The errors that the comments state are those of the constants as floats, in 64 bits."""
    source = (pkg._build.CSRC / "gdn_recurrence.cu").read_text()

    def constants(name):
        at = source.index(name + "[")
        text = source[source.index("{", at) + 1:source.index("}", at)]
        return [float(torch.tensor(float(v.strip().rstrip("f")))) for v in text.split(",")]

    def poly(c, x):
        return sum(k * x ** n for n, k in enumerate(c))

    u = torch.linspace(1e-4, 1, 1_000_001, dtype=torch.float64)
    log1p = float((poly(constants("kLog1p"), u) * u / torch.log1p(u) - 1).abs().max())
    t = torch.linspace(-0.25, 0, 1_000_001, dtype=torch.float64)
    exp2 = float(((1 + t * poly(constants("kExp2"), t)) / torch.exp2(t) - 1).abs().max())
    assert log1p <= 2.2e-7 and exp2 <= 3.7e-9
    assert "2.2e-7" in source and "3.7e-9" in source
