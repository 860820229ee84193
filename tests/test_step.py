"""The mixers' token step (``kdn_b200.decode``): T single-token calls against the
float64 oracle's whole-sequence operators (short convolution, gate frontend,
gain, memory recurrence, gated norm), which pins the step to the training
path's definitions.

Tolerance (normalised max-abs): the step computes in fp32 with sums of at most
128 terms (error below 128 * 2^-24 = 8e-6 of the sum's terms, in practice a
few 2^-24) and the decayed state does not amplify it, so 1e-5 for fp32
results; bf16 outputs carry one rounding more, 2^-9 of the value: 2^-8.
"""
import pytest
import torch

import oracle
from kdn_b200.decode import DiagKDNStep, IsoKDNStep, KDNState

OMEGA_MIN, R_MIN, EPS = 0.02, 0.01, 1e-5


def nmax(x, ref):
    x, ref = x.detach().double().cpu(), ref.detach().double().cpu()
    return ((x - ref).abs().max() / ref.abs().max().clamp_min(1e-30)).item()


def make(variant, B, T, H, D, dtype, seed=0):
    """CPU parameters and inputs of T tokens."""
    gen = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    HD = H * D
    p = {"conv_weight": n(3 * HD, 4) * 0.4, "A_log": n(H) * 0.5, "dt_bias": n(HD) * 0.5 - 1.0,
         "norm_weight": 1.0 + 0.2 * n(D), "prec": n(H)}
    x = {"qkv": n(B, T, 3 * HD).to(dtype), "decay": n(B, T, HD).to(dtype), "gate": n(B, T, HD).to(dtype)}
    if variant == "iso":
        p["omega_bias"], p["r_bias"] = 0.5 * n(H), 0.5 * n(H)
        x["omega_r"] = n(B, T, 2 * H).to(dtype)
    else:
        x["omega"], x["r"] = n(B, T, HD).to(dtype), n(B, T, H).to(dtype)
    return p, x


def truth(variant, p, x, H, D, activation="sigmoid", info_scale=None, with_norm=True):
    """(y [B, T, HD], memory, covariance) in float64."""
    p = {k: v.double() for k, v in p.items()}
    x = {k: v.double() for k, v in x.items()}
    B, T, _ = x["qkv"].shape
    q, k, v = oracle.short_conv(x["qkv"], p["conv_weight"]).view(B, T, 3, H, D).unbind(2)
    decay = x["decay"].view(B, T, H, D)
    if variant == "iso":
        _, a, omega, r, prec = oracle.iso_gate(decay, x["omega_r"], p["omega_bias"], p["r_bias"], p["A_log"],
                                               p["dt_bias"], p["prec"], OMEGA_MIN, R_MIN)
        log_alpha = -torch.exp(p["A_log"]).view(H, 1) * torch.nn.functional.softplus(decay + p["dt_bias"].view(H, D))
        alpha = torch.exp(log_alpha)
        beta, _, cov = oracle.iso_gain(a, omega, r, prec, 1.0 if info_scale is None else info_scale / D)
        q, k = oracle.l2norm(q), oracle.l2norm(k)
        kappa = beta[..., None] * k
    else:
        _, alpha, omega, r, prec = oracle.diag_gate(decay, x["omega"].view(B, T, H, D), x["r"], p["A_log"],
                                                    p["dt_bias"].view(H, D), p["prec"])
        q, k = (t / t.norm(dim=-1, keepdim=True).clamp_min(1e-12) for t in (q, k))
        kappa, cov = oracle.diag_gain(k, alpha, omega, r, prec)
        alpha = alpha.clamp_min(oracle.DIAG_ALPHA_FLOOR)
    S0 = torch.zeros(B, H, D, D, dtype=torch.float64)
    o, S = oracle.memory_recurrence(q, k, v, alpha, kappa, S0, D ** -0.5)
    w = p["norm_weight"] if with_norm else None
    y = oracle.rms_norm_gated(o, x["gate"].view(B, T, H, D), w, EPS, activation)
    return y.reshape(B, T, H * D), S, cov


def make_step(variant, p, activation="sigmoid", info_scale=None, with_norm=True):
    p = {k: v.cuda() for k, v in p.items()}
    shared = dict(norm_eps=EPS, activation=activation)
    w = p["norm_weight"] if with_norm else None
    if variant == "iso":
        return IsoKDNStep(p["conv_weight"], p["A_log"], p["dt_bias"], w, omega_bias=p["omega_bias"],
                          r_bias=p["r_bias"], omega_min=OMEGA_MIN, r_min=R_MIN, info_scale=info_scale, **shared)
    return DiagKDNStep(p["conv_weight"], p["A_log"], p["dt_bias"], w, **shared)


def token(variant, x, t):
    names = ("qkv", "decay", "omega_r", "gate") if variant == "iso" else ("qkv", "decay", "omega", "r", "gate")
    return [x[n][:, t] for n in names]


def initial_precision(p):
    return (0.1 + torch.nn.functional.softplus(p["prec"].double())).float()


@pytest.mark.gpu
@pytest.mark.parametrize("variant", ["iso", "diag"])
@pytest.mark.parametrize("B,H,D,dtype,slots", [(1, 18, 128, torch.bfloat16, None), (3, 1, 64, torch.float32, torch.int64),
                                               (13, 5, 128, torch.float32, torch.int32),
                                               (40, 7, 64, torch.bfloat16, torch.int32)])
def test_steps_match_oracle(variant, B, H, D, dtype, slots):
    T = 6
    p, x = make(variant, B, T, H, D, dtype, seed=B + H)
    y_ref, S_ref, cov_ref = truth(variant, p, x, H, D)
    step = make_step(variant, p)
    n = B if slots is None else B + 4
    state = KDNState.allocate(variant, n, H, D, dtype=dtype)
    index = None if slots is None else torch.randperm(n, generator=torch.Generator().manual_seed(1))[:B].cuda().to(slots)
    rows = torch.arange(B).cuda() if slots is None else index.long()
    others = torch.tensor([i for i in range(n) if i not in rows.tolist()], dtype=torch.long).cuda()
    # slots that are not in the call keep whatever they hold, NaN included
    state.memory[others], state.window[others] = float("nan"), 3.0
    state.covariance[others] = -1.0
    state.reset(rows, initial_precision(p).cuda())
    x = {k: v.cuda() for k, v in x.items()}
    ys = torch.stack([step(state, *(u.contiguous() for u in token(variant, x, t)), index) for t in range(T)], 1)
    assert ys.dtype == dtype
    assert nmax(ys, y_ref) < (2 ** -8 if dtype == torch.bfloat16 else 1e-5)
    assert nmax(state.memory[rows], S_ref) < 1e-5
    assert nmax(state.covariance[rows], cov_ref) < 1e-5
    assert torch.equal(state.window[rows], x["qkv"][:, -3:])
    assert state.memory[others].isnan().all() and (state.window[others] == 3.0).all()
    assert (state.covariance[others] == -1.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("variant", ["iso", "diag"])
def test_strided_rows_idle_rows_other_stream_and_options(variant):
    """Rows that are slices of one packed projection at an odd offset, rows marked idle, a stream of the caller's, the
    swish gate, no norm weight and (iso) an info scale."""
    B, T, H, D, dtype = 5, 3, 3, 128, torch.bfloat16
    p, x = make(variant, B, T, H, D, dtype, seed=9)
    info = 64 if variant == "iso" else None
    y_ref, S_ref, cov_ref = truth(variant, p, x, H, D, "swish", info, with_norm=False)
    step = make_step(variant, p, "swish", info, with_norm=False)
    state = KDNState.allocate(variant, B, H, D, dtype=dtype)
    state.reset(slice(None), initial_precision(p).cuda())
    before = state.memory.clone(), state.covariance.clone(), state.window.clone()
    idle = torch.tensor([False, True, False, False, True])
    slots = torch.tensor([0, -1, 2, 3, B], dtype=torch.int32).cuda()  # below and above the pool
    x = {k: v.cuda() for k, v in x.items()}
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    ys = []
    with torch.cuda.stream(stream):
        for t in range(T):
            parts = token(variant, x, t)
            packed = torch.cat([torch.zeros(B, 1, dtype=dtype, device="cuda"), *parts], 1)
            views = packed[:, 1:].split([u.shape[1] for u in parts], 1)
            ys.append(step(state, *views, slots))
    stream.synchronize()
    ys, live = torch.stack(ys, 1).cpu(), ~idle
    assert (ys[idle] == 0).all()
    assert nmax(ys[live], y_ref[live]) < 2 ** -8
    assert nmax(state.memory[live], S_ref[live]) < 1e-5
    assert nmax(state.covariance[live], cov_ref[live]) < 1e-5
    for now, old in zip((state.memory, state.covariance, state.window), before):
        assert torch.equal(now[idle], old[idle])


@pytest.mark.gpu
@pytest.mark.parametrize("variant", ["iso", "diag"])
def test_extreme_gates_and_zero_vectors(variant):
    """Decays that underflow (alpha = 0; the diagonal memory's floor), zero projections (|q| = |k| = 0) and large ones."""
    B, T, H, D = 4, 4, 2, 64
    p, x = make(variant, B, T, H, D, torch.float32, seed=4)
    x["decay"][0] = 300.0   # alpha underflows
    x["decay"][1] = -300.0  # alpha = 1
    x["qkv"][2] = 0.0
    x["qkv"][3] *= 100.0
    y_ref, S_ref, cov_ref = truth(variant, p, x, H, D)
    step = make_step(variant, p)
    state = KDNState.allocate(variant, B, H, D, dtype=torch.float32)
    state.reset(slice(None), initial_precision(p).cuda())
    x = {k: v.cuda() for k, v in x.items()}
    ys = torch.stack([step(state, *(u.contiguous() for u in token(variant, x, t))) for t in range(T)], 1)
    for b in range(B):
        assert nmax(ys[b], y_ref[b]) < 1e-5
        assert nmax(state.memory[b], S_ref[b]) < 1e-5
        assert nmax(state.covariance[b], cov_ref[b]) < 1e-5


@pytest.mark.gpu
def test_slot_beyond_32_bit_offsets():
    H, D, dtype = 18, 128, torch.bfloat16
    n = 2**31 // (H * D * D) + 2  # the last slots start past 2^31 elements (8.6 GB of states)
    p, x = make("iso", 1, 2, H, D, dtype, seed=2)
    y_ref, S_ref, _ = truth("iso", p, x, H, D)
    step = make_step("iso", p)
    state = KDNState(torch.empty(n, H, D, D, device="cuda"), torch.empty(n, H, device="cuda"),
                     torch.empty(n, 3, 3 * H * D, dtype=dtype, device="cuda"))
    state.reset([n - 1], initial_precision(p).cuda())
    slots = torch.tensor([n - 1], device="cuda")
    x = {k: v.cuda() for k, v in x.items()}
    ys = torch.stack([step(state, *(u.contiguous() for u in token("iso", x, t)), slots) for t in range(2)], 1)
    assert nmax(ys, y_ref) < 2 ** -8
    assert nmax(state.memory[n - 1:], S_ref) < 1e-5


@pytest.mark.gpu
@pytest.mark.parametrize("variant", ["iso", "diag"])
def test_continues_a_prompt_of_the_training_operators(variant):
    """A prompt through the chunked training operators (``sequence_parallel.*_segment``), then single tokens from the
    stored states, against the oracle over the whole sequence.  The prompt's kernels compute in bf16: the repository's
    scan tolerance 2e-2."""
    from kdn_b200.diag_kdn_chunk import _diag_kdn_frontend_precumsum_paired, _diag_kdn_normalize
    from kdn_b200.iso_kdn_chunk import _iso_kdn_gate_precumsum_paired
    from kdn_b200.sequence_parallel import diag_segment, iso_segment
    from kdn_b200.short_conv import qkv_causal_conv1d

    B, H, D, prompt, T, dtype = 2, 3, 128, 70, 75, torch.bfloat16
    p, x = make(variant, B, T, H, D, dtype, seed=7)
    y_ref, S_ref, cov_ref = truth(variant, p, x, H, D)
    pc, xc = {k: v.cuda() for k, v in p.items()}, {k: v.cuda() for k, v in x.items()}
    step = make_step(variant, p)
    state = KDNState.allocate(variant, B, H, D, dtype=dtype)
    head = {k: v[:, :prompt].contiguous() for k, v in xc.items()}
    with torch.no_grad():
        q, k, v = (t.view(B, prompt, H, D) for t in qkv_causal_conv1d(head["qkv"], pc["conv_weight"]))
        decay = head["decay"].view(B, prompt, H, D)
        if variant == "iso":
            g, a, w, r, prec = _iso_kdn_gate_precumsum_paired(
                decay, head["omega_r"], pc["omega_bias"], pc["r_bias"], pc["A_log"], pc["dt_bias"], pc["prec"],
                OMEGA_MIN, R_MIN)
            _, S, cov = iso_segment(q, k, v, g, a, w, r, prec)
        else:
            qm, kg, km = _diag_kdn_normalize(q, k)
            wr, rr = head["omega"].view(B, prompt, H, D), head["r"]
            g, alpha, w, r, prec = _diag_kdn_frontend_precumsum_paired(decay, wr, rr, pc["A_log"],
                                                                      pc["dt_bias"].view(H, D), pc["prec"])
            _, S, cov = diag_segment(qm, km, v, g, kg, alpha, w, r, prec, wr, rr)
    state.store(slice(None), S, cov, head["qkv"])
    ys = torch.stack([step(state, *(u.contiguous() for u in token(variant, xc, t))) for t in range(prompt, T)], 1)
    assert nmax(ys, y_ref[:, prompt:]) < 2e-2
    assert nmax(state.memory, S_ref) < 2e-2
    assert nmax(state.covariance, cov_ref) < 2e-2


@pytest.mark.gpu
def test_graph_capture_and_empty_batch():
    variant, B, H, D, dtype = "iso", 2, 2, 128, torch.bfloat16
    p, x = make(variant, B, 3, H, D, dtype, seed=3)
    step = make_step(variant, p)
    xs = [u.contiguous() for u in token(variant, {k: v.cuda() for k, v in x.items()}, 0)]
    state = KDNState.allocate(variant, B, H, D, dtype=dtype)
    state.reset(slice(None), initial_precision(p).cuda())
    first = state.memory.clone(), state.covariance.clone(), state.window.clone()
    want = [step(state, *xs) for _ in range(3)]
    end = state.memory.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step(state, *xs)
    for now, old in zip((state.memory, state.covariance, state.window), first):
        now.copy_(old)
    for w in want:
        graph.replay()
        assert torch.equal(y, w)
    assert torch.equal(state.memory, end)
    assert step(state, *(u[:0] for u in xs)).shape == (0, H * D)


def test_store_keeps_short_prompts_and_reset_starts_from_the_prior():
    state = KDNState.allocate("diag", 3, 2, 64, dtype=torch.float32, device="cpu")
    tail = torch.arange(2 * 2 * 384.0).view(2, 2, 384)
    state.store([2, 0], torch.ones(2, 2, 64, 64), torch.full((2, 2, 64), 5.0), tail)
    assert (state.window[2, 0] == 0).all() and torch.equal(state.window[2, 1:], tail[0])
    assert torch.equal(state.window[0, 1:], tail[1]) and (state.memory[1] == 0).all()
    state.reset([0], torch.tensor([2.0, 4.0]))
    assert (state.window[0] == 0).all() and (state.memory[0] == 0).all()
    assert torch.equal(state.covariance[0], torch.tensor([0.5, 0.25])[:, None].expand(2, 64))
    assert (state.covariance[2] == 5.0).all()


def test_refusals():
    f = torch.float32
    z = lambda *s, dtype=f: torch.zeros(*s, dtype=dtype)  # noqa: E731
    with pytest.raises(ValueError, match="memory must be"):
        KDNState(z(2, 3, 64, 32), z(2, 3), z(2, 3, 576))
    with pytest.raises(ValueError, match="D in"):
        KDNState(z(2, 3, 32, 32), z(2, 3), z(2, 3, 288))
    with pytest.raises(ValueError, match="covariance must be"):
        KDNState(z(2, 3, 64, 64), z(2, 4), z(2, 3, 576))
    with pytest.raises(ValueError, match="window must be"):
        KDNState(z(2, 3, 64, 64), z(2, 3), z(2, 4, 576))
    with pytest.raises(TypeError, match="FP32"):
        KDNState(z(2, 3, 64, 64, dtype=torch.bfloat16), z(2, 3), z(2, 3, 576))
    with pytest.raises(ValueError, match="contiguous"):
        KDNState(z(2, 3, 64, 128)[..., ::2], z(2, 3), z(2, 3, 576))
    H, D = 3, 64
    iso = dict(omega_bias=z(H), r_bias=z(H), omega_min=0.0, r_min=0.01)
    with pytest.raises(ValueError, match="conv_weight"):
        IsoKDNStep(z(3 * H * D, 3), z(H), z(H * D), None, **iso)
    with pytest.raises(ValueError, match="head dimension"):
        IsoKDNStep(z(3 * H * 48, 4), z(H), z(H * 48), None, **iso)
    with pytest.raises(ValueError, match="dt_bias"):
        IsoKDNStep(z(3 * H * D, 4), z(H), z(H), None, **iso)
    with pytest.raises(ValueError, match="activation"):
        IsoKDNStep(z(3 * H * D, 4), z(H), z(H * D), None, **iso, activation="relu")
    with pytest.raises(ValueError, match="info_scale"):
        IsoKDNStep(z(3 * H * D, 4), z(H), z(H * D), None, **iso, info_scale=-1.0)
    with pytest.raises(ValueError, match="finite"):
        IsoKDNStep(z(3 * H * D, 4), z(H), z(H * D), None, **{**iso, "r_min": float("nan")})
    step = IsoKDNStep(z(3 * H * D, 4), z(H), z(H * D), z(D), **iso)
    state = KDNState.allocate("iso", 2, H, D, dtype=f, device="cpu")
    good = [z(2, 3 * H * D), z(2, H * D), z(2, 2 * H), z(2, H * D)]

    def call(i=None, t=None, state=state, slots=None):
        step(state, *(t if j == i else u for j, u in enumerate(good)), slots)

    with pytest.raises(TypeError, match="variant"):
        call(state=KDNState.allocate("diag", 2, H, D, dtype=f, device="cpu"))
    with pytest.raises(ValueError, match="heads"):
        call(state=KDNState.allocate("iso", 2, 4, D, dtype=f, device="cpu"))
    with pytest.raises(ValueError, match="qkv must be"):
        call(0, z(2, H * D))
    with pytest.raises(TypeError, match="window"):
        call(0, good[0].bfloat16())
    with pytest.raises(ValueError, match="decay_raw must be"):
        call(1, z(3, H * D))
    with pytest.raises(ValueError, match="omega_r_raw must be"):
        call(2, z(2, H))
    with pytest.raises(TypeError, match="dtype"):
        call(3, good[3].double())
    with pytest.raises(ValueError, match="contiguous"):
        call(3, z(H * D, 2).t())
    with pytest.raises(ValueError, match="slots must be"):
        call(slots=torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError, match="slots must be"):
        call(slots=torch.zeros(2))
    with pytest.raises(ValueError, match="pool must hold"):
        call(state=KDNState.allocate("iso", 1, H, D, dtype=f, device="cpu"))
    if not torch.cuda.is_available():
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    else:
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_c_entry_refuses_without_launch():
    import ctypes

    from kdn_b200 import _native as N

    lib = N.load_library()
    assert lib.kdn_step(None, None) == -1 and b"null args" in lib.kdn_last_error()
    a = N.KdnStepArgs()
    a.variant, a.B, a.H, a.D = N.KDN_ISO, 1, 1, 96
    assert lib.kdn_step(a, None) == -1 and b"D in {64, 128}" in lib.kdn_last_error()
    a.D = 64
    assert lib.kdn_step(a, None) == -1 and b"null pointer" in lib.kdn_last_error()
    a.B, a.H = 1 << 40, 64
    assert lib.kdn_step(a, None) == -1 and b"too large" in lib.kdn_last_error()
    for name in ("qkv", "decay_raw", "omega_raw", "r_raw", "gate", "conv_weight", "A_log", "dt_bias", "omega_bias",
                 "r_bias", "covariance", "window", "y"):
        setattr(a, name, 16)
    a.B, a.H, a.num_slots, a.memory = 1, 1, 1, 8
    assert lib.kdn_step(a, None) == -1 and b"16-byte aligned" in lib.kdn_last_error()
    a.memory, a.num_slots = 16, 0
    assert lib.kdn_step(a, None) == -1 and b"pool must hold" in lib.kdn_last_error()
    a.B, a.num_slots, a.qkv_stride = 2, 2, 100  # neither 0 (one row for all) nor a whole row
    assert lib.kdn_step(a, None) == -1 and b"strides" in lib.kdn_last_error()
    assert ctypes.sizeof(N.KdnStepArgs) == 16 + 4 * 8 + 5 * 8 + 5 * 8 + 6 * 8 + 5 * 4 + 4 + 5 * 8
