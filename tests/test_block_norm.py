"""The norms around a block (``kdn_b200.block_norm``) against the formula in
float64 and its autograd, and against central differences.

Tolerances (normalised max-abs).  fp32 results: a row sum of up to 8192 terms
and a handful of roundings, a few 2^-24 each: 1e-5.  bf16 results: one rounding
more, 2^-9 of the value: 2^-8.  Weight gradients in fp32 sum up to 300 rows
here, in at most 300 sequential additions (300 * 2^-24 = 2e-5 of the terms in
the worst case, a few 1e-7 in practice): 2e-5.
"""
import pytest
import torch

from kdn_b200.block_norm import BlockNorm, block_norm

BF, F = torch.bfloat16, torch.float32
NAMES = ("x", "y", "gate", "weight", "post_weight", "scale")


def nmax(x, ref):
    x, ref = x.detach().double().cpu(), ref.detach().double().cpu()
    if not x.numel():
        return 0.0
    return ((x - ref).abs().max() / ref.abs().max().clamp_min(1e-30)).item()


def tol_of(t, weights=False):
    return 2 ** -8 if t.dtype == BF else 2e-5 if weights else 1e-5


def formula(x, y, gate, weight, post_weight, scale, alpha=1.0, activation="sigmoid", eps=1e-5):
    """(z, h) in the inputs' dtype (float64 in the tests)."""
    norm = lambda t: t / torch.sqrt((t * t).mean(-1, keepdim=True) + eps)  # noqa: E731
    z = x
    if y is not None:
        u = y
        if post_weight is not None:
            u = norm(u) * post_weight
        if gate is not None:
            s = torch.sigmoid(gate)
            u = u * (s if activation == "sigmoid" else gate * s)
        if scale is not None:
            u = u * scale
        z = alpha * x + u
    return z, norm(z) * weight


def make(shape, stream, dtype, parts="", wdtype=F, seed=0):
    """Inputs on CPU; parts: letters y (block), p (post norm), g (gate), s (scale)."""
    gen = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    D = shape[-1]
    return {"x": (2 * n(*shape)).to(stream), "y": n(*shape).to(dtype) if "y" in parts else None,
            "gate": n(*shape).to(dtype) if "g" in parts else None, "weight": (1 + 0.3 * n(D)).to(wdtype),
            "post_weight": (1 + 0.3 * n(D)).to(wdtype) if "p" in parts else None,
            "scale": (0.7 + 0.3 * n(D)).to(wdtype) if "s" in parts else None,
            "dz": n(*shape).to(stream), "dh": n(*shape).to(dtype)}


def reference(d, use=("dz", "dh"), **kw):
    leaves = {k: None if d[k] is None else d[k].double().requires_grad_(True) for k in NAMES}
    z, h = formula(**leaves, **kw)
    loss = sum((o * d[c].double()).sum() for o, c in ((z, "dz"), (h, "dh")) if c in use)
    loss.backward()
    return z, h, {k: v.grad for k, v in leaves.items() if v is not None and v.grad is not None}


def ours(d, use=("dz", "dh"), **kw):
    leaves = {k: None if d[k] is None else d[k].cuda().requires_grad_(True) for k in NAMES}
    z, h = block_norm(leaves["x"], leaves["y"], leaves["weight"], post_weight=leaves["post_weight"],
                      gate=leaves["gate"], scale=leaves["scale"], **kw)
    outs = [(o, d[c].cuda()) for o, c in ((z, "dz"), (h, "dh")) if c in use]
    torch.autograd.backward([o for o, _ in outs], [c for _, c in outs])
    return z, h, {k: v.grad for k, v in leaves.items() if v is not None and v.grad is not None}


def compare(d, **kw):
    z, h, grads = ours(d, **kw)
    zr, hr, gr = reference(d, **kw)
    assert z.dtype == d["x"].dtype and h.dtype == (d["x"] if d["y"] is None else d["y"]).dtype
    assert nmax(z, zr) < tol_of(z) and nmax(h, hr) < tol_of(h)
    assert set(grads) == set(gr)
    for k, g in grads.items():
        assert g.dtype == d[k].dtype and g.shape == d[k].shape
        assert nmax(g, gr[k]) < tol_of(g, k in NAMES[3:]), k


@pytest.mark.gpu
@pytest.mark.parametrize("parts", ["", "y", "yp", "yg", "ys", "ypgs"])
@pytest.mark.parametrize("stream,dtype", [(BF, BF), (F, BF), (F, F)])
@pytest.mark.parametrize("shape", [(3, 101, 2304), (7, 1155), (1, 64), (300, 40)])
def test_matches_formula(shape, stream, dtype, parts):
    dtype = dtype if "y" in parts else stream  # without a block, h has x's dtype
    compare(make(shape, stream, dtype, parts, seed=len(parts) + shape[-1]))


@pytest.mark.gpu
@pytest.mark.parametrize("D", [2, 7, 8, 255, 264, 2305, 4096, 4099, 8184, 8191, 8192])
@pytest.mark.parametrize("dtype", [BF, F])
def test_widths(D, dtype):
    compare(make((5, D), dtype, dtype, "ypgs", seed=D))


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [{"alpha": -0.5}, {"activation": "swish"}, {"eps": 0.3}])
def test_options(kw):
    compare(make((9, 200), F, F, "ypgs", seed=1), **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("use", [("dz",), ("dh",)])
@pytest.mark.parametrize("parts", ["y", "ypgs"])
def test_one_cotangent(parts, use):
    compare(make((9, 200), F, F, parts, seed=2), use=use)


@pytest.mark.gpu
def test_bf16_weights():
    compare(make((33, 136), BF, BF, "ypgs", wdtype=BF, seed=3))


@pytest.mark.gpu
@pytest.mark.parametrize("D", [96, 97])
def test_strided_and_unaligned_rows(D):
    """Rows that are slices of wider ones, at offsets that are not 16-byte aligned, and a transposed layout."""
    d = make((17, D), BF, BF, "ypgs", seed=4)
    want = {k: None if v is None else v.cuda() for k, v in d.items()}
    wide = torch.zeros(17, 3 * D + 5, dtype=BF, device="cuda")
    wide[:, 1:D + 1], wide[:, D + 2:2 * D + 2] = want["x"], want["y"]
    x, y = wide[:, 1:D + 1], wide[:, D + 2:2 * D + 2]
    gate = want["gate"].t().contiguous().t()
    kw = dict(post_weight=want["post_weight"], gate=gate, scale=want["scale"])
    z, h = block_norm(x, y, want["weight"], **kw)
    zr, hr = block_norm(want["x"], want["y"], want["weight"], **{**kw, "gate": want["gate"]})
    assert torch.equal(z, zr) and torch.equal(h, hr)
    zr, hr = formula(*(None if d[k] is None else d[k].double() for k in NAMES))
    assert nmax(z, zr) < 2 ** -8 and nmax(h, hr) < 2 ** -8


@pytest.mark.gpu
def test_saved_tensors_may_move():
    """Saved-tensor hooks that bring the tensors back elsewhere (activation offloading)."""
    d = make((5, 96), F, F, "ypgs", seed=12)
    _, _, want = ours(d)
    with torch.autograd.graph.save_on_cpu():
        leaves = {k: d[k].cuda().requires_grad_(True) for k in NAMES}
        z, h = block_norm(leaves["x"], leaves["y"], leaves["weight"], post_weight=leaves["post_weight"],
                          gate=leaves["gate"], scale=leaves["scale"])
    got = torch.autograd.grad((z, h), [leaves[k] for k in NAMES], (d["dz"].cuda(), d["dh"].cuda()))
    assert all(torch.equal(g, want[k]) for g, k in zip(got, NAMES))


@pytest.mark.gpu
def test_broadcast_gate():
    """One gate row for all rows (stride 0): the same outputs as its copies, and the sum of their gradients."""
    d = make((2, 6, 40), F, F, "yps", seed=9)
    x, y, w, p, s = (d[k].cuda() for k in ("x", "y", "weight", "post_weight", "scale"))
    row = torch.randn(40, device="cuda", requires_grad=True)
    copies = row.detach().expand(2, 6, 40).contiguous().requires_grad_(True)
    outs = []
    for gate in (row.expand(2, 6, 40), copies):
        z, h = block_norm(x, y, w, post_weight=p, gate=gate, scale=s)
        outs.append((z, h, torch.autograd.grad(h, row if gate is not copies else copies, d["dh"].cuda())[0]))
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])
    assert nmax(outs[0][2], outs[1][2].sum((0, 1))) < 1e-5
    z, h = block_norm(x, y, w, gate=row.detach().expand(2, 6, 40))
    zr, hr = formula(x.double(), y.double(), row.detach().double(), w.double(), None, None)
    assert nmax(z, zr) < 1e-5 and nmax(h, hr) < 1e-5


@pytest.mark.gpu
def test_empty_rows_zero_rows_and_large_values():
    d = make((0, 48), F, F, "ypgs")
    z, h, grads = ours(d)
    assert z.shape == h.shape == (0, 48)
    assert all((grads[k] == 0).all() and grads[k].shape == (48,) for k in NAMES[3:])
    d = make((4, 48), F, F, "ypgs", seed=5)
    d["x"][1], d["y"][1] = 0.0, 0.0  # norms of zero rows: eps alone
    d["x"][2] *= 1e15                # squares of the sum reach 1e32
    compare(d)


@pytest.mark.gpu
def test_repeats_exactly():
    d = make((301, 1000), BF, BF, "ypgs", seed=6)
    _, _, a = ours(d)
    _, _, b = ours(d)
    assert all(torch.equal(a[k], b[k]) for k in a)


@pytest.mark.gpu
@pytest.mark.parametrize("parts", ["", "y", "ypgs"])
def test_gradients_against_differences(parts):
    """Central differences of the kernel's own forward along random directions.  Step 2^-6: the outputs' rounding
    (99 values of order 1, 2^-24 each, summed in float64) moves the quotient by up to 99 * 2^-24 * 2^6 = 4e-4, the
    third derivative by about step^2 = 2.4e-4 times a factor of a few: 5e-3 of the scale of the derivative."""
    d = make((3, 33), F, F, parts, seed=8)
    _, _, grads = ours(d)
    gen = torch.Generator().manual_seed(1)
    step = 2.0 ** -6

    def loss(args):
        z, h = block_norm(args["x"], args["y"], args["weight"], post_weight=args["post_weight"], gate=args["gate"],
                          scale=args["scale"])
        return ((z.double() * d["dz"].cuda()).sum() + (h.double() * d["dh"].cuda()).sum()).item()

    for name in grads:
        base = {k: None if d[k] is None else d[k].cuda() for k in NAMES}
        direction = torch.randn(d[name].shape, generator=gen).cuda()
        up, down = dict(base), dict(base)
        up[name], down[name] = base[name] + step * direction, base[name] - step * direction
        slope = (loss(up) - loss(down)) / (2 * step)
        want = (grads[name].double() * direction).sum().item()
        size = grads[name].double().norm().item() * direction.double().norm().item()
        assert abs(slope - want) < 5e-3 * max(size, 1.0), name


@pytest.mark.gpu
def test_module_matches_function_and_other_streams():
    torch.manual_seed(0)
    mod = BlockNorm(72, post_norm=True, scale_init=0.1, alpha=2.0).cuda()
    x, y, gate = (torch.randn(2, 5, 72, device="cuda") for _ in range(3))
    z, h = mod(x, y, gate)
    zr, hr = block_norm(x, y, mod.weight, post_weight=mod.post_weight, gate=gate, scale=mod.scale, alpha=2.0)
    assert torch.equal(z, zr) and torch.equal(h, hr)
    z0, h0 = mod(x)
    assert z0 is x and torch.equal(h0, block_norm(x, None, mod.weight)[1])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        zs, hs = mod(x, y, gate)
    stream.synchronize()
    assert torch.equal(zs, z) and torch.equal(hs, h)


def test_refusals():
    x = torch.zeros(2, 8)
    w = torch.ones(8)
    with pytest.raises(ValueError, match="activation"):
        block_norm(x, x, w, activation="relu")
    with pytest.raises(ValueError, match="wide"):
        block_norm(torch.zeros(2, 8193), None, torch.ones(8193))
    with pytest.raises(ValueError, match="wide"):
        block_norm(torch.zeros(2, 0), None, torch.ones(0))
    with pytest.raises(ValueError, match="wide"):  # a norm over one value: refused (see the module)
        block_norm(torch.zeros(2, 1), None, torch.ones(1))
    with pytest.raises(TypeError, match="x must be"):
        block_norm(x.half(), None, w)
    with pytest.raises(ValueError, match="same shape"):
        block_norm(x, torch.zeros(3, 8), w)
    with pytest.raises(TypeError, match="dtype"):
        block_norm(x.bfloat16(), x, w)
    with pytest.raises(ValueError, match="need a block output"):
        block_norm(x, None, w, gate=x)
    with pytest.raises(ValueError, match="need a block output"):
        block_norm(x, None, w, alpha=0.5)
    with pytest.raises(ValueError, match="gate must"):
        block_norm(x, x, w, gate=x.bfloat16())
    with pytest.raises(ValueError, match="scale must"):
        block_norm(x, x, w, scale=torch.ones(7))
    with pytest.raises(TypeError, match="share one dtype"):
        block_norm(x, x, w, scale=w.bfloat16())
    with pytest.raises(TypeError, match="weight must be a tensor"):
        block_norm(x, x, None)
    if not torch.cuda.is_available():
        with pytest.raises(RuntimeError, match="CUDA"):
            block_norm(x, x, w)
    else:
        with pytest.raises(ValueError, match="CUDA"):
            block_norm(x, x, w)


def test_c_entry_refuses_without_launch():
    from kdn_b200 import _native as N

    lib = N.load_library()
    a = N.KdnBlockNormArgs()
    a.rows, a.D, a.alpha = 4, 1 << 15, 1.0
    assert lib.kdn_block_norm_fwd(a, None) == -1 and b"D in" in lib.kdn_last_error()
    a.D = 32
    assert lib.kdn_block_norm_fwd(a, None) == -1 and b"null pointer" in lib.kdn_last_error()
    a.x = a.weight = a.gate = 16
    a.x_stride = a.gate_stride = 32
    assert lib.kdn_block_norm_fwd(a, None) == -1 and b"need a block output" in lib.kdn_last_error()
    a.gate, a.x_stride = None, 31  # neither 0 nor a whole row
    assert lib.kdn_block_norm_fwd(a, None) == -1 and b"strides" in lib.kdn_last_error()
    a.x_stride, a.stream_bf16 = 32, 1
    assert lib.kdn_block_norm_fwd(a, None) == -1 and b"fp32 residual stream" in lib.kdn_last_error()
    a.stream_bf16, a.dweight = 0, 16
    assert lib.kdn_block_norm_bwd(a, None) == -1 and b"rstd" in lib.kdn_last_error()
    a.rstd = 16
    assert lib.kdn_block_norm_bwd(a, None) == -2 and b"workspace" in lib.kdn_last_error()
    a.dscale = 16
    assert lib.kdn_block_norm_bwd(a, None) == -1 and b"absent input" in lib.kdn_last_error()
    assert lib.kdn_block_norm_workspace_bytes(4, 32) > 0 and lib.kdn_block_norm_workspace_bytes(0, 32) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("D", [3, 36, 97, 1155])
@pytest.mark.parametrize("stream,dtype", [(BF, BF), (F, F)])
def test_rows_do_not_touch_their_neighbours(D, stream, dtype):
    """Rows that share 16-byte words of memory: what one of them holds changes nothing in the others, and an output
    row ends where the next begins."""
    d = make((21, D), stream, dtype, "ypgs", seed=D)
    z, h, grads = ours(d)
    for k in ("x", "y", "gate", "dz", "dh"):
        d[k] = d[k].clone()
        d[k][7], d[k][12] = float("nan"), float("inf")
    zn, hn, spoilt = ours(d)
    rest = [i for i in range(21) if i not in (7, 12)]
    for a, b in ((z, zn), (h, hn), *((grads[k], spoilt[k]) for k in ("x", "y", "gate"))):
        assert torch.equal(a[rest], b[rest]) and not b[7].isfinite().any()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 2, 9, 1201])
@pytest.mark.parametrize("D", [10, 100, 801])
def test_few_and_many_odd_rows(rows, D):
    compare(make((rows, D), F, F, "ypgs", seed=rows + D))


def loose(t, offset=1, gap=2):
    """t's rows as slices of wider ones, `offset` values behind a 16-byte boundary, NaN around them."""
    wide = torch.full((t.shape[0], t.shape[1] + offset + gap), float("nan"), dtype=t.dtype, device=t.device)
    view = wide[:, offset:offset + t.shape[1]]
    view.copy_(t)
    return view


def check_loose(d, lay, **kw):
    """Outputs and every gradient against the formula; lay: how a CPU tensor [rows, D] goes to the GPU."""
    leaves = {}
    for k in NAMES:
        if d[k] is not None:
            leaves[k] = (lay(k, d[k]) if d[k].ndim == 2 else d[k].cuda()).detach().requires_grad_(True)
    get = leaves.get
    z, h = block_norm(get("x"), get("y"), get("weight"), post_weight=get("post_weight"), gate=get("gate"),
                      scale=get("scale"), **kw)
    zr, hr, gr = reference(d, **kw)
    assert nmax(z, zr) < tol_of(z) and nmax(h, hr) < tol_of(h)
    grads = torch.autograd.grad((z, h), list(leaves.values()), (d["dz"].cuda(), d["dh"].cuda()))
    for k, g in zip(leaves, grads):
        assert g.dtype == d[k].dtype and g.shape == d[k].shape
        assert nmax(g, gr[k]) < tol_of(g, k in NAMES[3:]), k


@pytest.mark.gpu
@pytest.mark.parametrize("D", [2, 3, 5, 7])
@pytest.mark.parametrize("stream,dtype", [(BF, BF), (F, BF), (F, F)])
def test_narrow_strides(D, stream, dtype):
    """Rows that start less than 16 bytes apart: the words that cover a row reach past its neighbours."""
    check_loose(make((37, D), stream, dtype, "ypgs", seed=D), lambda k, t: loose(t.cuda(), 1, 0))


@pytest.mark.gpu
@pytest.mark.parametrize("D", [3, 97, 1155])
@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("offset", [0, 1, 5])
def test_one_odd_row_for_all(D, dtype, offset):
    """Stride 0 at odd widths and offsets, NaN on both sides of the one row."""
    d = make((11, D), dtype, dtype, "ypgs", seed=D + offset)
    for k in ("x", "gate"):
        d[k] = d[k][:1].expand(11, D)
    check_loose(d, lambda k, t: loose(t[:1].cuda(), offset).expand(11, D) if k in ("x", "gate") else t.cuda())


@pytest.mark.gpu
@pytest.mark.parametrize("D,many", [(3, 8000), (97, 8000), (1155, 5000), (4099, 700), (8191, 700)])
@pytest.mark.parametrize("stream,dtype", [(BF, BF), (F, BF), (F, F)])
@pytest.mark.parametrize("parts,few", [("y", True), ("ypgs", True), ("ypgs", False), ("pygs", False)])
def test_loose_rows_match_formula(D, many, stream, dtype, parts, few):
    """Outputs and gradients of rows with odd strides and offsets (cotangents too): few, and more than the CTAs hold at a
    time.  Weight gradients: the sums of up to 8000 random terms have partial sums of the order of the result, added in
    some 50 steps, 50 * 2^-24 = 3e-6 of it: 2e-5."""
    rows = 5 if few else many
    offsets = {"x": 1, "y": 3, "gate": 2} if parts == "ypgs" else {"x": 0, "y": 1, "gate": 7}
    d = make((rows, D), stream, dtype, parts, seed=D + rows)
    leaves = {k: None if d[k] is None else (loose(d[k].cuda(), offsets[k]) if k in offsets else d[k].cuda())
              .detach().requires_grad_(True) for k in NAMES}

    def packed(t):  # contiguous, one value behind a 16-byte boundary
        room = torch.full((t.numel() + 1,), float("nan"), dtype=t.dtype, device="cuda")
        room[1:] = t.cuda().flatten()
        return room[1:].view(t.shape)

    z, h = block_norm(leaves["x"], leaves["y"], leaves["weight"], post_weight=leaves["post_weight"], gate=leaves["gate"],
                      scale=leaves["scale"])
    zr, hr, gr = reference(d)
    assert nmax(z, zr) < tol_of(z) and nmax(h, hr) < tol_of(h)
    names = [k for k in NAMES if leaves[k] is not None]
    grads = torch.autograd.grad((z, h), [leaves[k] for k in names], (packed(d["dz"]), packed(d["dh"])))
    for k, g in zip(names, grads):
        assert g.dtype == d[k].dtype and g.shape == d[k].shape
        assert nmax(g, gr[k]) < tol_of(g, k in NAMES[3:]), k
