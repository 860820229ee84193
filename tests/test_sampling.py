"""Token sampling (``kdn_b200.sampling.sample``) against its definition in
float64.

Tokens must be equal.  The kernel's sums and quotients are fp32 (relative
error below 2^-20 for the sums of up to 2^17 positive terms here), so a row is
compared only where the float64 token is clear: the race's two best scores are
1e-5 apart, and moving top_p and min_p by 1e-5 up or down leaves the token.
At most 2% of a case's rows may be left out for that.  prob is compared at
1e-5 relative.
"""
import math

import numpy as np
import pytest
import torch

from kdn_b200.sampling import sample

MARGIN = 1e-5


def truth(logits, noise, temperature, top_k, top_p, min_p):
    """(token, prob, clear) of one row in float64; clear: the token stands within the margin."""
    l = np.where(np.isnan(logits), -np.inf, logits.astype(np.float64))
    top = l.max()
    if top == -np.inf:
        return -1, 0.0, True
    order = np.lexsort((np.arange(l.size), -l))
    if not temperature > 0:
        return int(order[0]), 1.0, True
    with np.errstate(invalid="ignore", divide="ignore"):
        e = np.where(l == top, 1.0, np.exp((l - top) / float(np.float32(temperature))))[order]
    Z = e.sum()
    winners, best = set(), None
    for slack in (0.0, -MARGIN, MARGIN):  # the filters' sums and thresholds, and both ends of their margin
        n = e.size if top_k is None or top_k <= 0 else min(int(top_k), e.size)
        if top_p is not None and top_p < 1:
            before = np.concatenate(([0.0], np.cumsum(e)[:-1]))
            n = min(n, int((before < (float(np.float32(top_p)) + slack) * Z).sum()))
        if min_p is not None:
            n = min(n, int((e >= float(np.float32(min_p)) * (1 - slack)).sum()))
        n = max(n, 1)
        kept = e[:n] > 0
        kept[0] = True
        with np.errstate(divide="ignore"):
            score = np.where(kept, e[:n] / noise[order[:n]].astype(np.float64), -1.0)
        win = int(np.argmax(score))
        winners.add(win)
        best = win if best is None else best
        if kept.sum() > 1 and not score[win] > np.partition(score, -2)[-2] * (1 + MARGIN):
            winners.add(-1)  # the race itself is too close
    return int(order[best]), e[best] / Z, len(winners) == 1


def check(logits, noise, rows_out=0.02, **options):
    dev = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in options.items()}
    token, prob = sample(logits.cuda(), noise.cuda(), **dev)
    assert token.dtype == torch.int64 and prob.dtype == torch.float32
    token, prob = token.cpu(), prob.cpu()
    get = lambda name, default, i: (default if options.get(name) is None else  # noqa: E731
                                    options[name][i].item() if isinstance(options[name], torch.Tensor)
                                    else options[name])
    unclear = 0
    for i in range(logits.shape[0]):
        want, p, clear = truth(logits[i].float().numpy(), noise[i].numpy(), get("temperature", 1.0, i),
                               get("top_k", None, i), get("top_p", None, i), get("min_p", None, i))
        if not clear:
            unclear += 1
            continue
        assert token[i] == want, (i, token[i].item(), want)
        assert abs(prob[i].item() - p) <= 1e-5 * p, i
    assert unclear <= max(1, rows_out * logits.shape[0]), unclear
    return token, prob


def make(rows, V, dtype=torch.bfloat16, spread=3.0, seed=0):
    gen = torch.Generator().manual_seed(seed)
    logits = (torch.randn(rows, V, generator=gen) * spread).to(dtype)
    return logits, torch.empty(rows, V).exponential_(generator=gen)


@pytest.mark.gpu
@pytest.mark.parametrize("V", [1, 2, 31, 1024, 1025, 5003, 32000, 131072])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_unfiltered(V, dtype):
    check(*make(6, V, dtype, seed=V))


@pytest.mark.gpu
@pytest.mark.parametrize("V,rows", [(17, 200), (1000, 200), (32000, 24), (100003, 8)])
@pytest.mark.parametrize("options", [{"top_k": 1}, {"top_k": 40}, {"top_k": 3000}, {"top_p": 0.9}, {"top_p": 0.2},
                                     {"top_p": 1e-9}, {"min_p": 0.05}, {"top_k": 50, "top_p": 0.8, "min_p": 0.01},
                                     {"temperature": 0.3, "top_p": 0.97}, {"temperature": 5.0, "top_k": 7}])
def test_filters(V, rows, options):
    check(*make(rows, V, seed=V + len(options)), **options)


@pytest.mark.gpu
@pytest.mark.parametrize("spread", [0.02, 1.0, 30.0])
def test_flat_and_peaked_rows_with_mixed_parameters(spread):
    rows, V = 96, 9001
    logits, noise = make(rows, V, torch.float32, spread, seed=int(spread * 10))
    gen = torch.Generator().manual_seed(5)
    u = lambda: torch.rand(rows, generator=gen)  # noqa: E731
    check(logits, noise, rows_out=0.05, temperature=torch.where(u() < 0.2, 0.0, 0.4 + u()),
          top_k=torch.where(u() < 0.4, 0, (u() * 300).int()).int(), top_p=torch.where(u() < 0.4, 1.0, u()),
          min_p=torch.where(u() < 0.5, 0.0, 0.2 * u()))


@pytest.mark.gpu
@pytest.mark.parametrize("options", [{}, {"top_k": 5}, {"top_p": 0.55}, {"min_p": 0.5}])
def test_ties_masks_infinities_and_nan(options):
    """Equal logits rank by index; -inf, the type's lowest value and NaN are never drawn beside others; +inf wins."""
    rows, V = 12, 700
    logits, noise = make(rows, V, torch.float32, seed=11)
    logits[0] = 0.25                                   # everything equal
    logits[1] = -math.inf                              # nothing left
    logits[2] = math.nan
    logits[3] = -math.inf
    logits[3, 699] = -2.0                              # one left
    logits[4, 10::7] = math.nan
    logits[5] = torch.finfo(torch.float32).min         # every token at the lowest value: an even draw
    logits[6] = torch.finfo(torch.float32).min
    logits[6, 333] = -50.0
    logits[7, [5, 600]] = math.inf                     # two certain tokens
    logits[8] = (logits[8] * 2).round()                # few distinct values
    logits[9, 1:] = -math.inf
    logits[10] = logits[10].abs() * -1e30
    noise[11] = 1.0                                    # no randomness: the first of the order
    token, prob = check(logits, noise, **options)
    assert token[1] == token[2] == -1 and prob[1] == prob[2] == 0
    assert token[3] == 699 and prob[3] == 1 and token[7] in (5, 600) and prob[7] == 0.5 and token[9] == 0
    assert not torch.isnan(prob).any()


@pytest.mark.gpu
def test_extreme_noise():
    logits, _ = make(4, 300, seed=3)
    noise = torch.ones(4, 300)
    noise[0, 17] = 0.0           # an infinite score
    noise[1] = math.inf          # every score 0: the first of the order
    noise[2] = 1e-38
    token, _ = sample(logits.cuda(), noise.cuda())
    assert token[0] == 17 and token[1] == logits[1].float().argmax() and token[2] == logits[2].float().argmax()
    noise[3] = math.nan          # not a random number: still a token of the row
    token, _ = sample(logits.cuda(), noise.cuda(), top_k=3)
    assert 0 <= token[3] < 300


@pytest.mark.gpu
def test_extreme_parameters():
    """Temperatures from below the fp32 range of 1 / T to infinity, thresholds outside [0, 1]: always a token of the
    row, and the most likely one where the definition leaves no other."""
    V = 3000
    logits, noise = make(1, V, torch.float32, seed=21)
    first = logits[0].argmax().item()
    T = torch.tensor([0.0, -1.0, math.nan, 1e-45, 1e-38, 1e-36, 1e-20, 1e-3])
    token, prob = sample(logits.expand(8, V).cuda(), noise.expand(8, V).cuda(), temperature=T.cuda())
    assert (token == first).all() and (prob == 1).all()
    token, prob = sample(logits.cuda(), noise.cuda(), temperature=math.inf)  # an even draw
    assert token[0] == (1 / noise[0]).argmax() and abs(prob[0].item() * V - 1) < 1e-5
    for options in ({"top_p": 0.0}, {"top_p": -1.0}, {"min_p": 1.5}, {"min_p": math.inf}, {"top_k": 1, "top_p": 0.0}):
        token, _ = sample(logits.cuda(), noise.cuda(), **options)
        assert token[0] == first, options
    for options in ({"top_p": 2.0}, {"top_p": math.inf}, {"min_p": -1.0}, {"top_k": -3}, {"top_k": V + 1}):
        assert torch.equal(sample(logits.cuda(), noise.cuda(), **options)[0], sample(logits.cuda(), noise.cuda())[0])


@pytest.mark.gpu
@pytest.mark.parametrize("options", [{}, {"top_k": 4}, {"top_p": 0.7}])
def test_winner_always_last_of_the_order(options):
    """Noise that favours the rear of the order at every turn, so that every race is lost to a later token."""
    V = 20000
    logits = torch.linspace(3.0, -3.0, V).repeat(2, 1)
    logits[1] = logits[1].flip(0)
    e = torch.exp(logits.double() - 3.0)
    noise = (e * e).float()  # score 1 / e grows towards the rear
    check(logits, noise, rows_out=0.0, **options)


@pytest.mark.gpu
def test_strides_other_stream_and_repeats():
    logits, noise = make(5, 999, seed=6)
    wide_l = torch.zeros(5, 2001, dtype=torch.bfloat16, device="cuda")
    wide_n = torch.ones(5, 1502, device="cuda")
    wide_l[:, 3:1002], wide_n[:, 1:1000] = logits.cuda(), noise.cuda()
    want, _ = check(logits, noise, top_p=0.9)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        outs = [sample(wide_l[:, 3:1002], wide_n[:, 1:1000], top_p=0.9) for _ in range(3)]
    stream.synchronize()
    for token, prob in outs:
        assert torch.equal(token.cpu(), want) and torch.equal(prob, outs[0][1])
    token, prob = sample(logits.cuda()[:0], noise.cuda()[:0])
    assert token.shape == prob.shape == (0,)


@pytest.mark.gpu
def test_top_k_types_and_whole_batch_values():
    logits, noise = make(7, 500, seed=8)
    k = torch.tensor([1, 2, 3, 0, -5, 500, 10**6])
    a, _ = check(logits, noise, top_k=k)
    b, _ = check(logits, noise, top_k=k.int())
    assert torch.equal(a, b)


@pytest.mark.gpu
def test_frequencies():
    """60000 draws of one distribution: each kept token's share within 5 standard deviations of its probability."""
    rows, V = 60000, 12
    l = torch.linspace(1.5, -1.5, V).repeat(rows, 1)
    noise = torch.empty(rows, V).exponential_(generator=torch.Generator().manual_seed(12))
    token, _ = sample(l.cuda(), noise.cuda(), temperature=0.8, top_k=6)
    p = torch.exp(l[0, :6].double() / 0.8)
    p /= p.sum()
    share = torch.bincount(token.cpu(), minlength=V).double() / rows
    assert (share[6:] == 0).all()
    assert ((share[:6] - p).abs() < 5 * torch.sqrt(p * (1 - p) / rows)).all()


def test_refusals():
    l, n = torch.zeros(2, 5), torch.ones(2, 5)
    with pytest.raises(ValueError, match="logits must be"):
        sample(l[0], n[0])
    with pytest.raises(ValueError, match="logits must be"):
        sample(l[:, :0], n[:, :0])
    with pytest.raises(TypeError, match="logits must be"):
        sample(l.half(), n)
    with pytest.raises(ValueError, match="noise must be"):
        sample(l, n[:1])
    with pytest.raises(ValueError, match="noise must be"):
        sample(l, n.double())
    with pytest.raises(ValueError, match="contiguous"):
        sample(torch.zeros(5, 2).t(), n)
    with pytest.raises(ValueError, match="temperature must be"):
        sample(l, n, temperature=torch.ones(3))
    with pytest.raises(ValueError, match="top_k must be"):
        sample(l, n, top_k=torch.ones(2))
    with pytest.raises(TypeError, match="top_p must be"):
        sample(l, n, top_p="all")
    with pytest.raises(ValueError, match="min_p must be"):
        sample(l, n, min_p=torch.ones(2, dtype=torch.float64))
    if not torch.cuda.is_available():
        with pytest.raises(RuntimeError, match="CUDA"):
            sample(l, n)
    else:
        with pytest.raises(ValueError, match="CUDA"):
            sample(l, n)


def test_c_entry_refuses_without_launch():
    from kdn_b200 import _native as N

    lib = N.load_library()
    assert lib.kdn_sample(None, None) == -1
    a = N.KdnSampleArgs()
    a.rows, a.V = 2, 0
    assert lib.kdn_sample(a, None) == -1 and b"V" in lib.kdn_last_error()
    a.V = 10
    assert lib.kdn_sample(a, None) == -1 and b"null pointer" in lib.kdn_last_error()
    a.logits = a.noise = a.token = a.prob = 16
    a.logits_stride = 9
    assert lib.kdn_sample(a, None) == -1 and b"strides" in lib.kdn_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,V", [(torch.bfloat16, 800000), (torch.bfloat16, 786433), (torch.float32, 400003)])
@pytest.mark.parametrize("options", [{}, {"top_k": 1}, {"top_k": 2000}, {"top_p": 0.6}, {"temperature": 0.0},
                                     {"top_k": 300, "top_p": 0.9, "min_p": 0.001}])
def test_rows_beyond_shared_memory(dtype, V, options):
    """Vocabularies of which eight CTAs of 192 KB do not hold a row: the rest is read again in every pass.  Winners and
    kept tokens among that rest, rows that start on 16-byte boundaries and rows that do not."""
    held, chunk = 192 * 1024 // dtype.itemsize, (V + 63) // 64 * 8
    rest = torch.arange(V) % chunk >= held
    assert rest.any()
    wide, wide_n = V + 8 - V % 8 + 8, V + 4 - V % 4 + 4  # row strides of whole 16-byte words
    logits, noise = make(3, V, dtype, 2.0, seed=V)
    logits[1, rest] += 6.0
    logits[2, ~rest] = -math.inf
    want, _ = check(logits, noise, **options)
    assert rest[want[2]]
    for shift in (0, 3):
        l = torch.full((3, wide), 50.0, dtype=dtype, device="cuda")
        n = torch.full((3, wide_n), 1e-9, device="cuda")
        l[:, shift:shift + V], n[:, shift:shift + V] = logits.cuda(), noise.cuda()
        for i in (slice(None), slice(1, 2)):
            token, _ = sample(l[i, shift:shift + V], n[i, shift:shift + V], **options)
            assert torch.equal(token.cpu(), want[i])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [700, 1501, 40000])
@pytest.mark.parametrize("options", [{"temperature": 0.0}, {}, {"top_k": 3}, {"top_p": 0.6}, {"min_p": 0.5}])
def test_nan_beside_infinity(dtype, V, options):
    """NaN logits count as -inf in rows with +inf too, whichever comes first."""
    logits, noise = make(3, V, dtype, seed=V)
    logits[:, ::3] = math.nan
    logits[0, [1, 640]] = math.inf
    logits[1, [4, 5, 695]] = math.inf
    logits[2, 698] = math.inf
    token, _ = check(logits, noise, **options)
    assert token[2] == 698


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1e20, 1e32, math.inf])
@pytest.mark.parametrize("options", [{}, {"top_k": 9}, {"top_p": 0.4937}])
def test_hot_rows(T, options):
    """Temperatures beside which the logits' differences are small, whatever their size: finite masks and large logits
    are drawn with their weight, -inf never."""
    logits, noise = make(8, 900, torch.float32, seed=4)
    logits[:, ::2] = torch.finfo(torch.float32).min
    logits[1] = logits[1].clamp(-1, 1) * 1e32
    logits[2] = -math.inf
    logits[2, 100:] = -1e31
    logits[3, 5::7] = -math.inf
    token, prob = sample(logits.cuda(), noise.cuda(), temperature=T, **options)
    unclear = 0
    for i in range(8):  # the definition over the tokens above -inf: exp(-inf / T) is 0, also where T is infinite
        at = torch.nonzero(logits[i] > -math.inf)[:, 0]
        want, p, clear = truth(logits[i, at].numpy(), noise[i, at].numpy(), T, options.get("top_k"), options.get("top_p"),
                               None)
        if not clear:
            unclear += 1
            continue
        assert token[i].item() == at[want], i
        assert abs(prob[i].item() - p) <= 1e-5 * p, i
    assert unclear <= 1


@pytest.mark.gpu
def test_whole_batch_top_k_beyond_64_bits():
    logits, noise = make(64, 500, seed=30)
    l, n = logits.cuda(), noise.cuda()
    want, _ = sample(l, n)
    for k in (2**31, 2**63, 2**64 + 1, 10**30, -2**64 + 1):
        assert torch.equal(sample(l, n, top_k=k)[0], want), k
    with pytest.raises(TypeError, match="top_k must be"):
        sample(l, n, top_k=math.inf)


@pytest.mark.gpu
@pytest.mark.parametrize("options", [{}, {"top_p": 0.9}, {"top_k": 50, "top_p": 0.8}])
def test_rows_alone_and_in_a_batch(options):
    """A row is cut into more parts when few rows are in the call: its sum Z then differs by rounding (positive terms,
    some 100 additions one after another: 100 * 2^-24 = 6e-6), its token only where that decides."""
    logits, noise = make(64, 32000, seed=3)
    token, prob = check(logits, noise, **options)
    differ = 0
    for i in range(64):
        t, p = check(logits[i:i + 1], noise[i:i + 1], **options)
        if t[0] == token[i]:
            assert abs(p[0] - prob[i]) <= 6e-6 * prob[i]
        else:
            differ += 1
    assert differ <= 1
