"""The two host paths of the serving operators (``csrc/host/kdn_torch.cpp`` and the Python one behind it) make the
same C calls: equal outputs, gradients and refusals."""
import contextlib
import os

import pytest
import torch

from kdn_b200 import _native as N
from kdn_b200.block_norm import block_norm
from kdn_b200.decode import DiagKDNStep, IsoKDNStep, KDNState
from kdn_b200.sampling import sample


@contextlib.contextmanager
def python_path():
    kept, N._host = N._host, False
    try:
        yield
    finally:
        N._host = kept


def both(call):
    """The call's tensors by the C++ path and by the Python path."""
    if N.host() is None:
        pytest.skip("the C++ host path is not built")
    first = call()
    with python_path():
        assert N.host() is None
        second = call()
    return first, second


def equal(a, b):
    assert len(a) == len(b)
    for x, y in zip(a, b):
        assert (x is None) == (y is None)
        if x is not None:
            assert x.dtype == y.dtype and x.shape == y.shape and torch.equal(x, y)


def test_the_build_has_it():
    import os

    from kdn_b200 import build

    build.build()
    assert os.path.exists(build.HOST_LIB)
    assert N.host() is not None


@pytest.mark.gpu
@pytest.mark.parametrize("parts", ["", "g", "ps", "pgs"])
@pytest.mark.parametrize("shape,strided", [((6, 40), False), ((2, 3, 96), False), ((5, 33), True)])
@pytest.mark.parametrize("needs", ["xygwps", "xw", "g", ""])
def test_block_norm(parts, shape, strided, needs):
    gen = torch.Generator().manual_seed(3)
    D = shape[-1]

    def tensor(name, *s):
        t = torch.randn(*s, generator=gen).cuda()
        if strided and len(s) > 1:
            wide = torch.zeros(s[0], s[1] + 3, device="cuda")
            wide[:, 1:-2] = t
            t = wide[:, 1:-2]
        return t.detach().requires_grad_(name in needs)

    x, y, w = tensor("x", *shape), tensor("y", *shape), tensor("w", D)
    g = tensor("g", *shape) if "g" in parts else None
    p, s = (tensor(n, D) if n in parts else None for n in "ps")
    leaves = [t for t in (x, y, g, w, p, s) if t is not None and t.requires_grad]
    cz, ch = torch.randn(*shape, generator=gen).cuda(), torch.randn(*shape, generator=gen).cuda()

    def call():
        z, h = block_norm(x, y, w, post_weight=p, gate=g, scale=s, activation="swish", alpha=0.5)
        out = [z, h]
        if leaves:
            out += torch.autograd.grad((z, h), leaves, (cz, ch), allow_unused=True, retain_graph=True)
            out += torch.autograd.grad(z, leaves, cz, allow_unused=True)
        return [t if t is None else t.detach() for t in out]

    equal(*both(call))


@pytest.mark.gpu
def test_block_norm_twice_differentiated_is_an_error():
    x, y, w = (torch.randn(*s, device="cuda", requires_grad=True) for s in ((3, 16), (3, 16), (16,)))

    def call():
        z, h = block_norm(x, y, w)
        (gx,) = torch.autograd.grad(h.square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiate twice"):
            gx.sum().backward()
        return [gx.detach()]

    equal(*both(call))


@pytest.mark.gpu
@pytest.mark.parametrize("variant", ["iso", "diag"])
@pytest.mark.parametrize("slots", [None, torch.int32, torch.int64])
def test_step(variant, slots):
    B, H, D = 3, 2, 64
    gen = torch.Generator().manual_seed(5)
    n = lambda *s: torch.randn(*s, generator=gen).cuda()  # noqa: E731
    shared = dict(conv_weight=n(3 * H * D, 4), A_log=n(H), dt_bias=n(H * D), norm_weight=n(D))
    if variant == "iso":
        step = IsoKDNStep(**shared, omega_bias=n(H), r_bias=n(H), omega_min=0.0, r_min=0.01)
        widths = (3 * H * D, H * D, 2 * H, H * D)
    else:
        step = DiagKDNStep(**shared)
        widths = (3 * H * D, H * D, H * D, H, H * D)
    packed = n(B, sum(widths) + 1)
    views = packed[:, 1:].split(widths, 1)
    index = None if slots is None else torch.tensor([2, -1, 0], dtype=slots, device="cuda")

    def call():
        state = KDNState.allocate(variant, 4, H, D, dtype=torch.float32)
        state.reset(slice(None), torch.ones(H, device="cuda"))
        ys = [step(state, *views, index) for _ in range(3)]
        return [*ys, state.memory, state.covariance, state.window]

    equal(*both(call))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_sample(dtype):
    gen = torch.Generator().manual_seed(6)
    logits, noise = torch.randn(7, 1001, generator=gen).to(dtype).cuda(), torch.empty(7, 1001).exponential_(generator=gen).cuda()
    k = torch.tensor([1, 5, 0, 50, 1000, 3, 2])
    for options in ({}, {"top_k": 7}, {"top_k": k.cuda()}, {"top_k": k.int().cuda(), "temperature": 0.5},
                    {"top_p": 0.9, "min_p": torch.full((7,), 0.01, device="cuda")}, {"temperature": 0},
                    {"temperature": torch.linspace(0, 1, 7, device="cuda"), "top_p": 1}):
        equal(*both(lambda: sample(logits, noise, **options)))


@pytest.mark.gpu
def test_refusals_are_the_same():
    x, w = torch.zeros(2, 8, device="cuda"), torch.ones(8, device="cuda")
    calls = [lambda: block_norm(x, x[:, :7], w), lambda: block_norm(x.bfloat16(), x, w), lambda: block_norm(x, x, w[:7]),
             lambda: block_norm(x, x, w, gate=x.bfloat16()), lambda: block_norm(x, x, w, scale=w.cpu()),
             lambda: block_norm(x, x, w, activation="relu"), lambda: block_norm(x, x, None),
             lambda: sample(x, x, top_k="five"), lambda: sample(x, x[:1]), lambda: sample(x, x, temperature=w),
             lambda: sample(x, x, temperature=None)]
    for call in calls:
        errors = []
        for path in (contextlib.nullcontext, python_path):
            with path(), pytest.raises((ValueError, TypeError)) as e:
                call()
            errors.append((e.type, str(e.value)))
        assert errors[0] == errors[1]


@pytest.mark.gpu
@pytest.mark.parametrize("path", [contextlib.nullcontext, python_path])
@pytest.mark.parametrize("which", ["x", "y", "weight", "post_weight", "gate", "scale"])
@pytest.mark.parametrize("grad", [True, False])
def test_block_norm_refuses_forward_mode_derivatives(path, which, grad):
    from torch.autograd import forward_ad

    args = {k: torch.randn(*((5, 40) if k in ("x", "y", "gate") else (40,)), device="cuda")
            for k in ("x", "y", "weight", "post_weight", "gate", "scale")}
    with path(), torch.set_grad_enabled(grad), forward_ad.dual_level():
        args[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(NotImplementedError, match="jvp"):
            block_norm(**args)
        if which in ("x", "weight"):  # without a block
            with pytest.raises(NotImplementedError, match="jvp"):
                block_norm(args["x"], None, args["weight"])
    with path(), forward_ad.dual_level():  # a level without tangents changes nothing
        plain = {k: forward_ad.unpack_dual(v).primal for k, v in args.items()}
        z, _ = block_norm(**plain)
    assert torch.equal(z, block_norm(**plain)[0])


@pytest.mark.gpu
@pytest.mark.parametrize("path", [contextlib.nullcontext, python_path])
@pytest.mark.parametrize("variant,which", [("iso", i) for i in range(4)] + [("diag", i) for i in range(5)])
def test_step_says_that_it_has_no_derivative(path, variant, which):
    from torch.autograd import forward_ad

    B, H, D = 2, 2, 64
    gen = torch.Generator().manual_seed(7)
    n = lambda *s: torch.randn(*s, generator=gen).cuda()  # noqa: E731
    shared = dict(conv_weight=n(3 * H * D, 4).requires_grad_(True), A_log=n(H), dt_bias=n(H * D), norm_weight=n(D))
    if variant == "iso":
        step = IsoKDNStep(**shared, omega_bias=n(H), r_bias=n(H), omega_min=0.0, r_min=0.01)
        widths = (3 * H * D, H * D, 2 * H, H * D)
    else:
        step = DiagKDNStep(**shared)
        widths = (3 * H * D, H * D, H * D, H, H * D)
    token = [n(B, w) for w in widths]

    def run():
        state = KDNState.allocate(variant, B, H, D, dtype=torch.float32)
        state.reset(slice(None), torch.ones(H, device="cuda"))
        return step(state, *token)

    with path():
        want = run()
        assert not want.requires_grad
        token[which].requires_grad_(True)
        y = run()
        assert torch.equal(y, want)
        with pytest.raises(RuntimeError, match="no gradient"):
            y.sum().backward()
        with torch.no_grad():
            y = run()
        assert torch.equal(y, want) and not y.requires_grad
        with torch.no_grad(), forward_ad.dual_level():
            token[which] = forward_ad.make_dual(token[which].detach(), torch.ones_like(token[which]))
            state = KDNState.allocate(variant, B, H, D, dtype=torch.float32)
            with pytest.raises(NotImplementedError, match="jvp"):
                step(state, *token)
            assert not state.window.any()  # refused before anything has happened


@pytest.mark.gpu
@pytest.mark.parametrize("path", [contextlib.nullcontext, python_path])
def test_block_norm_of_overlapping_rows(path):
    """A sliding window over one line of values: rows closer together than they are long."""
    D = 40
    line = torch.randn(200, device="cuda")
    x, y, gate = line.unfold(0, D, 1)[:50], line.unfold(0, D, 3)[:50], line[100:].unfold(0, D, 1)[:50]
    w = torch.rand(D, device="cuda")
    want = block_norm(x.contiguous(), y.contiguous(), w, gate=gate.contiguous())
    with path():
        equal(block_norm(x, y, w, gate=gate), want)
        h = block_norm(x, None, w)[1]
        assert torch.equal(h, block_norm(x.contiguous(), None, w)[1])
        leaf = line.clone().requires_grad_(True)
        z, _ = block_norm(leaf.unfold(0, D, 1)[:50], y, w)
        (g,) = torch.autograd.grad(z.sum(), leaf)
    hits = torch.zeros(200, device="cuda").index_add_(0, torch.arange(200, device="cuda").unfold(0, D, 1)[:50].flatten(),
                                                      torch.ones(50 * D, device="cuda"))
    assert torch.equal(g, hits)


def test_host_library_of_another_torch_or_broken(tmp_path, monkeypatch):
    """Never loaded, one warning, and the Python path."""
    import warnings

    from kdn_b200 import build

    assert torch.__version__ in os.path.basename(build.HOST_LIB)
    monkeypatch.delenv("KDN_B200_HOST", raising=False)
    ours = tmp_path / "_kdn_torch.2.0.abi.so"
    monkeypatch.setattr(N, "HOST_LIB", str(ours))
    for name, match in (("_kdn_torch.1.9.abi.so", "another torch"), (ours.name, "does not load")):
        (tmp_path / name).write_bytes(b"not a library")
        monkeypatch.setattr(N, "_host", None)
        with pytest.warns(UserWarning, match=match):
            assert N.host() is None
        with warnings.catch_warnings():
            warnings.simplefilter("error")
            assert N.host() is None


def test_build_without_a_host_compiler(tmp_path, monkeypatch):
    from kdn_b200 import build

    stale = tmp_path / "_kdn_torch.so"
    stale.write_bytes(b"of an older source")
    kernels = []
    monkeypatch.setattr(build, "HOST_LIB", str(stale))
    monkeypatch.setattr(build, "up_to_date", lambda: False)
    monkeypatch.setattr(build, "host_up_to_date", lambda: False)
    monkeypatch.setattr(build, "_build_kernels", lambda verbose: kernels.append(1))
    monkeypatch.setattr(build, "_nvcc", lambda: "/usr/local/cuda/bin/nvcc")
    monkeypatch.setenv("PATH", str(tmp_path))
    with pytest.warns(UserWarning, match="host path is not built"):
        assert build.build() == build.LIB
    assert kernels and not stale.exists()
    monkeypatch.setattr(build, "host_up_to_date", lambda: True)

    def fails(verbose):
        raise RuntimeError("nvcc failed")

    monkeypatch.setattr(build, "_build_kernels", fails)
    with pytest.raises(RuntimeError, match="nvcc failed"):  # the kernels are needed
        build.build()
