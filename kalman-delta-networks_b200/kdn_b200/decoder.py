"""A small KDN language model that trains and generates on this package's
operators: an example of how they are used together.

    x = embedding                                     residual stream
    per layer:  x, h = norm(x, ...);  mixer(h);  x, h = norm(x, mixer output);  SwiGLU MLP(h)
    logits = head(norm(x, last MLP output))

* Training and prompts (:meth:`KDNDecoder.forward`): the chunked operators (short convolution, gate frontend, gain,
  memory scan, gated norm) over whole sequences, and ``block_norm`` between the blocks.
* Generation (:meth:`KDNDecoder.generate`): the prompt leaves its states in a :class:`~kdn_b200.decode.KDNState` per
  layer; every further token is one ``kdn_step`` per layer, ``block_norm`` between the blocks and ``sample`` at the end,
  replayed as one CUDA graph.

The projections are plain matrix products.  Run it with random weights:

    python -m kdn_b200.decoder --variant iso --layers 2 --heads 4 --prompt 100 --tokens 32
"""
from __future__ import annotations

import argparse

import torch
import torch.nn as nn
import torch.nn.functional as F

from .block_norm import BlockNorm
from .decode import DIAG_R_MIN, DiagKDNStep, IsoKDNStep, KDNState
from .diag_kdn_chunk import _diag_kdn_frontend_precumsum_paired, _diag_kdn_normalize
from .iso_kdn_chunk import _iso_kdn_gate_precumsum_paired
from .norm_gated import rms_norm_gated
from .sampling import sample
from .sequence_parallel import diag_segment, iso_segment
from .short_conv import GROUPS, KERNEL_WIDTH, qkv_causal_conv1d

HEAD_DIM = 128
OMEGA_MIN, R_MIN, NORM_EPS = 0.0, DIAG_R_MIN, 1e-5


class KDNMixer(nn.Module):
    """One KDN mixer (isotropic or diagonal); ``forward`` over sequences, ``step`` for one token."""

    def __init__(self, variant, hidden, heads, device=None, dtype=torch.bfloat16):
        super().__init__()
        if variant not in ("iso", "diag"):
            raise ValueError(f"variant must be 'iso' or 'diag', got {variant!r}")
        self.variant, self.heads = variant, heads
        channels = heads * HEAD_DIM
        # q | k | v, decay, omega, r, output gate: one projection
        self.widths = [GROUPS * channels, channels, *((2 * heads,) if variant == "iso" else (channels, heads)), channels]
        self.in_proj = nn.Linear(hidden, sum(self.widths), bias=False, device=device, dtype=dtype)
        self.out_proj = nn.Linear(channels, hidden, bias=False, device=device, dtype=dtype)
        new = lambda *s: nn.Parameter(torch.empty(*s, device=device))  # noqa: E731
        self.conv_weight = new(GROUPS * channels, KERNEL_WIDTH)
        self.A_log, self.dt_bias, self.norm_weight = new(heads), new(channels), new(HEAD_DIM)
        self.prior = new(heads)  # the initial precision before its softplus
        self.omega_bias, self.r_bias = (new(heads), new(heads)) if variant == "iso" else (None, None)
        with torch.no_grad():
            nn.init.uniform_(self.conv_weight, -0.5, 0.5)
            self.A_log.copy_(torch.log(torch.linspace(1.0, 8.0, heads)))
            self.dt_bias.fill_(-4.0)
            self.norm_weight.fill_(1.0)
            for p in (self.prior, self.omega_bias, self.r_bias):
                if p is not None:
                    p.zero_()

    def forward(self, h):
        """h [B, T, hidden] -> (output [B, T, hidden], states: memory, covariance, the last rows of q | k | v)."""
        B, T, _ = h.shape
        H, D = self.heads, HEAD_DIM
        parts = [t.contiguous() for t in self.in_proj(h).split(self.widths, -1)]
        qkv, decay, gate = parts[0], parts[1].view(B, T, H, D), parts[-1].view(B, T, H, D)
        q, k, v = (t.view(B, T, H, D) for t in qkv_causal_conv1d(qkv, self.conv_weight))
        if self.variant == "iso":
            g, a, omega, r, prec = _iso_kdn_gate_precumsum_paired(
                decay, parts[2], self.omega_bias, self.r_bias, self.A_log, self.dt_bias, self.prior, OMEGA_MIN, R_MIN)
            o, memory, covariance = iso_segment(q, k, v, g, a, omega, r, prec)
        else:
            q_mem, k_gain, k_mem = _diag_kdn_normalize(q, k)
            omega_raw, r_raw = parts[2].view(B, T, H, D), parts[3]
            g, alpha, omega, r, prec = _diag_kdn_frontend_precumsum_paired(
                decay, omega_raw, r_raw, self.A_log, self.dt_bias.view(H, D), self.prior)
            o, memory, covariance = diag_segment(q_mem, k_mem, v, g, k_gain, alpha, omega, r, prec, omega_raw, r_raw)
        y = rms_norm_gated(o.to(h.dtype), gate, self.norm_weight, activation="sigmoid", eps=NORM_EPS)
        return self.out_proj(y.reshape(B, T, H * D)), (memory, covariance, qkv[:, -(KERNEL_WIDTH - 1):])

    def make_step(self):
        shared = dict(conv_weight=self.conv_weight, A_log=self.A_log, dt_bias=self.dt_bias, norm_weight=self.norm_weight,
                      norm_eps=NORM_EPS)
        if self.variant == "iso":
            return IsoKDNStep(**shared, omega_bias=self.omega_bias, r_bias=self.r_bias, omega_min=OMEGA_MIN, r_min=R_MIN)
        return DiagKDNStep(**shared)

    def step(self, kdn_step, state, h, slots):
        """h [B, hidden], one token per row -> [B, hidden]; the projection's slices go to the kernel as they are."""
        qkv, *parts = self.in_proj(h).split(self.widths, -1)
        return self.out_proj(kdn_step(state, qkv, *parts, slots))


class SwiGLU(nn.Module):
    def __init__(self, hidden, inner, device=None, dtype=torch.bfloat16):
        super().__init__()
        self.up = nn.Linear(hidden, 2 * inner, bias=False, device=device, dtype=dtype)
        self.down = nn.Linear(inner, hidden, bias=False, device=device, dtype=dtype)

    def forward(self, h):
        a, b = self.up(h).chunk(2, -1)
        return self.down(F.silu(a) * b)


class KDNDecoder(nn.Module):
    """``layers`` KDN blocks over a vocabulary.  post_norm and scale_init: norms after the blocks and a learned residual
    scale (``BlockNorm``); the residual stream is fp32 or bf16 (``stream``)."""

    def __init__(self, vocab, hidden, layers, heads, *, variant="iso", inner=None, post_norm=False, scale_init=None,
                 stream=torch.float32, device="cuda", dtype=torch.bfloat16):
        super().__init__()
        self.vocab, self.stream, self.dtype = vocab, stream, dtype
        inner = 4 * hidden if inner is None else inner
        self.embedding = nn.Embedding(vocab, hidden, device=device, dtype=dtype)
        self.mixers = nn.ModuleList(KDNMixer(variant, hidden, heads, device, dtype) for _ in range(layers))
        self.mlps = nn.ModuleList(SwiGLU(hidden, inner, device, dtype) for _ in range(layers))
        # norms[0] is in front of the first block, norms[i + 1] joins sublayer i's output and comes before the next
        self.norms = nn.ModuleList([BlockNorm(hidden, device=device)] + [
            BlockNorm(hidden, post_norm=post_norm, scale_init=scale_init, device=device) for _ in range(2 * layers)])
        self.head = nn.Linear(hidden, vocab, bias=False, device=device, dtype=dtype)

    def _blocks(self, tokens, mix):
        """The last norm's output; mix(layer, h) runs a mixer."""
        x, h = self.norms[0](self.embedding(tokens).to(self.stream))
        for i, mlp in enumerate(self.mlps):
            x, h = self.norms[2 * i + 1](x, mix(i, h.to(self.dtype)))
            x, h = self.norms[2 * i + 2](x, mlp(h))
        return h

    def forward(self, tokens, states=None):
        """tokens [B, T] -> logits [B, T, vocab]; with a list ``states``, appends every layer's states to it."""
        def mix(i, h):
            out, state = self.mixers[i](h)
            if states is not None:
                states.append(state)
            return out

        return self.head(self._blocks(tokens, mix))

    @torch.no_grad()
    def start(self, prompts, pools, slots):
        """Run prompts [n, T] and leave their states at ``slots`` of every layer's pool; returns the last logits [n, vocab]."""
        states = []
        logits = self.forward(prompts, states)[:, -1]
        for pool, (memory, covariance, tail) in zip(pools, states):
            pool.store(slots, memory, covariance, tail)
        return logits

    def make_pools(self, num_slots):
        mixer = self.mixers[0]
        return [KDNState.allocate(mixer.variant, num_slots, mixer.heads, HEAD_DIM, dtype=self.dtype,
                                  device=self.embedding.weight.device) for _ in self.mixers]

    @torch.no_grad()
    def decode(self, tokens, pools, steps, slots=None):
        """One token per row: tokens [B] -> logits [B, vocab]; the pools advance."""
        return self.head(self._blocks(tokens, lambda i, h: self.mixers[i].step(steps[i], pools[i], h, slots)))

    @torch.no_grad()
    def generate(self, prompts, count, *, generator=None, graph=True, **options):
        """``count`` tokens after every row of prompts [B, T]; options as :func:`~kdn_b200.sampling.sample` takes them.
        Returns (tokens [B, count], their probabilities [B, count]); -1 and 0 where a row's logits are all NaN or -inf."""
        if prompts.ndim != 2 or prompts.shape[1] < 1:
            raise ValueError(f"prompts must be [B, T] with T >= 1, got {tuple(prompts.shape)}")
        if count < 0:
            raise ValueError(f"count must not be negative, got {count}")
        B = prompts.shape[0]
        if count == 0:
            return prompts.new_empty((B, 0), dtype=torch.int64), prompts.new_empty((B, 0), dtype=torch.float32)
        pools, steps = self.make_pools(B), [m.make_step() for m in self.mixers]
        slots = torch.arange(B, dtype=torch.int32, device=prompts.device)
        logits = self.start(prompts, pools, slots.long())
        noise = torch.empty(B, self.vocab, device=prompts.device)
        draw = lambda: noise.exponential_(generator=generator).clamp_(min=1e-30)  # noqa: E731
        draw()
        new, prob = sample(logits, noise, **options)
        tokens, probs = [new.clone()], [prob.clone()]
        token = new.clamp(min=0)  # a row that lost its numbers (token -1) goes on with token 0: the embedding has no row -1

        def advance():
            return sample(self.decode(token, pools, steps, slots), noise, **options)

        replay = None
        for i in range(1, count):
            draw()
            if not graph or i < 3:  # the first calls set the kernels up; a graph starts after them
                new, p = advance()
            else:
                if replay is None:
                    replay = torch.cuda.CUDAGraph()
                    with torch.cuda.graph(replay):  # records only
                        new, p = advance()
                replay.replay()
            torch.clamp(new, min=0, out=token)
            tokens.append(new.clone())
            probs.append(p.clone())
        return torch.stack(tokens, 1), torch.stack(probs, 1)


def main():
    ap = argparse.ArgumentParser(description="Generate tokens with a randomly initialised KDN decoder.")
    ap.add_argument("--variant", choices=("iso", "diag"), default="iso")
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--heads", type=int, default=4)
    ap.add_argument("--vocab", type=int, default=1000)
    ap.add_argument("--batch", type=int, default=4)
    ap.add_argument("--prompt", type=int, default=100)
    ap.add_argument("--tokens", type=int, default=32)
    ap.add_argument("--temperature", type=float, default=0.8)
    ap.add_argument("--top-k", type=int, default=50)
    ap.add_argument("--top-p", type=float, default=0.95)
    ap.add_argument("--seed", type=int, default=0)
    a = ap.parse_args()
    torch.manual_seed(a.seed)
    model = KDNDecoder(a.vocab, a.heads * HEAD_DIM, a.layers, a.heads, variant=a.variant)
    prompts = torch.randint(a.vocab, (a.batch, a.prompt), device="cuda")
    generator = torch.Generator(device="cuda").manual_seed(a.seed)
    options = dict(temperature=a.temperature, top_k=a.top_k, top_p=a.top_p)
    model.generate(prompts, 4, **options)  # loads the kernels
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    begin.record()
    tokens, probs = model.generate(prompts, a.tokens, generator=generator, **options)
    end.record()
    torch.cuda.synchronize()
    for row, p in zip(tokens.tolist(), probs.tolist()):
        print(" ".join(f"{t}({q:.2f})" for t, q in zip(row, p)))
    print(f"{begin.elapsed_time(end):.1f} ms for {a.batch} prompts of {a.prompt} tokens and {a.tokens} new tokens each")


if __name__ == "__main__":
    main()


__all__ = ("KDNDecoder", "KDNMixer", "SwiGLU")
