"""Decoding over a paged cache end to end: bounded decoding against a plain loop in 64 bits that keeps each layer's rows as lists, bfloat16 logits
against the dense cache's on the same ids, and drafted samples against the target's own distribution."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def _model(seed, E=128, H=4, L=2, stablemax=False, sharp=6.0):
    """A random model whose attention is uneven (queries and keys scaled up): what a slot holds and where it was matters."""
    from multimodal_amd.models import MultiModalToSMILESModel
    torch.manual_seed(seed)
    m = MultiModalToSMILESModel(591, 1000, max_seq_length=40, max_nmr_length=16, max_memory_length=32, embed_dim=E, num_heads=H, num_layers=L,
                                dropout=0.0, verbose=False, use_stablemax=stablemax)
    with torch.no_grad():
        for l in m.decoder.layers:
            l.q.weight.mul_(sharp); l.k.weight.mul_(sharp)
        m.decoder.out.weight.mul_(8)
    return m.to(DEV).eval()


def _inputs(B, seed=5):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(0, 1000, (B, 16), generator=g).to(DEV), torch.rand(B, 1000, generator=g).to(DEV)


class Plain:
    """The decoder in 64 bits on the host, from its formulas: per layer K (rotated), V [B, H, n, d] and accumulated weights [B, H, n], grown
    by concatenation."""

    def __init__(self, dec, prompt):
        self.dec, self.H = dec, dec.num_heads
        self.par = {k: v.detach().double().cpu() for k, v in dec.state_dict().items()}
        x = prompt.double().cpu()
        B, self.P, _ = x.shape
        self.k, self.v, self.w = [], [], []
        for l in range(len(dec.layers)):
            q, k, v = self.project(l, x, torch.arange(self.P))
            self.k.append(k); self.v.append(v); self.w.append(torch.zeros(k.shape[:3], dtype=torch.float64))
            x = self.rest(l, x, self.weigh(q, k) @ v)

    def lin(self, x, name):
        return x @ self.par[name + ".weight"].t() + self.par[name + ".bias"]

    def norm(self, x, name):
        x = x - x.mean(-1, keepdim=True)
        return x / (x.square().mean(-1, keepdim=True) + 1e-5).sqrt() * self.par[name + ".weight"] + self.par[name + ".bias"]

    def project(self, l, x, pos):
        """x [B, n, E] at positions pos [n]: q, k rotated in the half layout, v, as [B, H, n, d]."""
        n, p = f"layers.{l}.", self.norm(x, f"layers.{l}.attn_norm")
        q, k, v = (self.lin(p, n + c).unflatten(-1, (self.H, -1)).transpose(1, 2) for c in "qkv")
        layer = self.dec.layers[l]
        a = pos[:, None].double() * layer.rotary_emb.inv_freq.double().cpu()
        c, s, h = a.cos(), a.sin(), layer.rotary_ndims // 2
        turn = lambda y: torch.cat((y[..., :h] * c - y[..., h:2 * h] * s, y[..., h:2 * h] * c + y[..., :h] * s, y[..., 2 * h:]), -1)
        return turn(q), turn(k), v

    def weigh(self, q, k):
        x = q @ k.transpose(-1, -2) / math.sqrt(q.shape[-1])
        if not self.dec.layers[0].use_stablemax:
            return torch.softmax(x, -1)
        s = torch.where(x < 0, 1 / (1 - x + 1e-9), x + 1)
        return s / s.sum(-1, keepdim=True).clamp_min(1e-9)

    def rest(self, l, x, o):
        n = f"layers.{l}."
        x = x + self.lin(o.transpose(1, 2).flatten(2), n + "out")
        return x + self.lin(self.lin(self.norm(x, n + "mlp_norm"), n + "ffn_w1").clamp(min=0).square(), n + "ffn_w2")

    def step(self, ids, pos):
        """One token of every row at position pos: logits [B, V]."""
        x = self.par["smiles_embed.weight"][ids.cpu()][:, None]
        for l in range(len(self.k)):
            q, k, v = self.project(l, x, torch.tensor([pos]))
            self.k[l], self.v[l] = torch.cat((self.k[l], k), 2), torch.cat((self.v[l], v), 2)
            p = self.weigh(q, self.k[l])
            self.w[l] = torch.cat((self.w[l], torch.zeros_like(self.w[l][..., :1])), 2) + p[:, :, 0]
            x = self.rest(l, x, p @ self.v[l])
        return self.lin(self.norm(x[:, 0], "final_norm"), "out")

    def evict(self, l, kept, recent, slack):
        """kept [B, H, budget] has to be the newest slots and, by these weights (ties within slack), the heaviest of the others; drops the rest."""
        kept = kept.long().cpu()
        n, A = self.w[l].shape[-1], kept.shape[-1] - recent
        assert (kept[..., A:] == torch.arange(n - recent, n)).all()
        chosen = torch.zeros_like(self.w[l], dtype=torch.bool).scatter_(2, kept, True)
        assert (chosen.sum(-1) == kept.shape[-1]).all()
        old = torch.arange(n) < n - recent
        least = self.w[l].masked_fill(~chosen | ~old, math.inf).amin(-1)
        most = self.w[l].masked_fill(chosen, -math.inf).amax(-1)
        assert (least >= most - slack).all(), float((most - least).max())
        pick = lambda x: x.gather(2, kept[..., None].expand(*kept.shape, x.shape[-1]))
        self.k[l], self.v[l], self.w[l] = pick(self.k[l]), pick(self.v[l]), self.w[l].gather(2, kept)


@pytest.mark.parametrize("stablemax", [False, True])
@pytest.mark.parametrize("budget,recent", [(30, 6), (50, 3), (20, 20)])
def test_bounded_decoding_against_a_plain_loop(monkeypatch, budget, recent, stablemax):
    """Every step's logits, one to eleven evictions long, and every eviction's choice.  Tolerance, float32: a product or a norm adds at most
    512 + 2 roundings of 2^-24 to what the step's largest value is; two layers have 12 of them with the output's: 12 * 514 * 2^-24."""
    import multimodal_amd as mm
    from multimodal_amd import generate as G, ops
    m = _model(3, stablemax=stablemax)
    nmr, ir = _inputs(5)
    steps, events = 36, []
    step, evict = G._PagedDecoder.step, ops.paged_evict

    def spy_step(self, ids, positions=None):
        out = step(self, ids, positions)
        events.append(("step", ids.clone(), out.clone()))
        return out

    def spy_evict(*a, **k):
        kept = evict(*a, **k)
        events.append(("evict", kept.clone()))
        return kept
    monkeypatch.setattr(G._PagedDecoder, "step", spy_step)
    monkeypatch.setattr(ops, "paged_evict", spy_evict)
    with mm.compute_dtype(torch.float32):
        got = m.generate(nmr, ir, max_len=steps, early_stop=False, page_size=8, kv_budget=budget, kv_recent=recent)
        plain = Plain(m.decoder, m.decoder.build_prompt(m.encoder(None, ir, None), nmr, torch.float32).detach())
    tol = 12 * 514 * 2.0 ** -24
    t = cuts = 0
    for e in events:
        if e[0] == "step":
            assert torch.equal(e[1], got[:, t])
            want = plain.step(e[1], plain.P + t)
            assert float((e[2].double().cpu() - want).abs().max()) <= tol * float(want.abs().max()), t
            t += 1
            layer = 0
        else:
            plain.evict(layer, e[1], recent, tol * t)                          # weights: t probabilities, each within the tolerance of 1
            layer += 1; cuts += layer == 2
    limit = max(budget, plain.P) + recent - plain.P                            # the tokens before the first eviction; every `recent` from then on
    assert t == steps and cuts == 1 + (steps - limit) // recent


@pytest.mark.parametrize("stablemax", [False, True])
def test_bf16_logits_of_the_paged_and_the_dense_step(stablemax):
    """The same ids through both caches (prompt keys rotated in place and copied, the same keys and values appended).  Both round at the same
    16 places (7 a layer, 2 for the output), by up to 2^-8 each: the dense step's distance from the plain loop stays below 16 * 2^-8 of the
    logits' length over all steps.  The paged step's distance is another draw of the same errors: at most twice the dense one over all
    steps, four times in a single one.  (A position off by one moves these logits by 4 to 13 %, prompt keys without their rotation by 7 to 23.)"""
    import multimodal_amd as mm
    from multimodal_amd import functional as FN, generate as G, ops
    m = _model(4, stablemax=stablemax, sharp=3.0)
    dec, (nmr, ir) = m.decoder, _inputs(6)
    B, steps, dt = 6, 24, torch.bfloat16
    ids = torch.randint(0, 591, (steps, B), generator=torch.Generator().manual_seed(1)).to(DEV)
    far = {"dense": [], "paged": []}
    with torch.no_grad(), mm.compute_dtype(dt):
        pd = G._PagedDecoder(m, nmr, ir, lambda P: P + steps, steps, 16)
        prompt = dec.build_prompt(m.encoder(None, ir, None), nmr, dt)
        plain = Plain(dec, prompt)
        P, E, H = pd.P, dec.embed_dim, dec.num_heads
        Smax = P + steps
        cache, weights = G.KVCache(len(dec.layers), B, H, Smax, E // H, dt, DEV), [G._layer_weights(l, dt) for l in dec.layers]
        G._prefill(dec, weights, prompt, Smax, lambda li, k, v, rot, c, s: ops.kv_cache_fill(k, v, cache.k[li], cache.v[li], H, rot, c, s))
        for t in range(steps):
            def attend(li, layer, qkv):
                return ops.decode_attn(qkv[:, :E], qkv[:, E:2 * E], qkv[:, 2 * E:], cache.k[li], cache.v[li], H, layer.rotary_ndims, P + t,
                                       *layer.rotary_emb.half_tables(Smax), layer.use_stablemax)
            h = dec.smiles_embed.weight[ids[t]].to(dt)
            dense = G._rows_logits(dec, weights, h, attend, FN.cached_operand((dec.out.weight,), dt), dec.out.bias.detach(),
                                   FN.cached_operand((dec.out.bias,), dt))
            paged = pd.step(ids[t])
            pd.cache.lengths.add_(1)
            want = plain.step(ids[t], P + t)
            for name, x in (("dense", dense), ("paged", paged)):
                far[name].append(float((x.double().cpu() - want).norm() / want.norm()))
    dense, paged = (torch.tensor(far[x]) for x in ("dense", "paged"))
    rms = lambda x: float(x.square().mean().sqrt())
    print(f"distance from the plain loop: dense {rms(dense):.4f} paged {rms(paged):.4f}, largest step {float(dense.max()):.4f} {float(paged.max()):.4f}")
    assert rms(dense) <= 16 * 2.0 ** -8
    assert rms(paged) <= 2 * rms(dense) and float(paged.max()) <= 4 * rms(dense)


def _drafting_pair():
    """A target, and a draft with its output weights disturbed: about half of the drafts are accepted."""
    m, d = _model(21, E=64, H=2, L=1), _model(21, E=64, H=2, L=1)
    with torch.no_grad():
        w = d.decoder.out.weight
        w.add_(torch.randn(w.shape, generator=torch.Generator().manual_seed(0)).to(DEV) * w.std() * 0.6)
    return m, d


@pytest.mark.parametrize("n_draft", [1, 2, 4])
def test_drafted_samples_are_distributed_as_the_target(monkeypatch, n_draft):
    """8192 rows of one spectrum: the first three tokens (the second and third behind the most frequent ones before them) occur as often as the
    target's softmax says.  A count over N rows leaves |count / N - p| <= sqrt(2 p (1 - p) c / N) + 2 c / (3 N) with probability at most
    2 exp(-c) (Bernstein); c is such that all of the test's 3 * 591 counts together leave it with 10^-9."""
    import multimodal_amd as mm
    from multimodal_amd import generate as G, ops
    N, T, temperature, V = 8192, n_draft + 1, 1.5, 591
    m, d = _drafting_pair()
    nmr, ir = (x.expand(N, -1).contiguous() for x in _inputs(1))
    calls, verify = [], ops.verify_drafts

    def spy(drafts, p, u, q=None, counts=None):
        out = verify(drafts, p, u, q=q, counts=counts)
        calls.append((drafts, p, u, q, out[0], out[1]))
        return out
    monkeypatch.setattr(ops, "verify_drafts", spy)
    with torch.no_grad(), mm.compute_dtype(torch.float32):
        got = G.speculative_generate(m, d, nmr, ir, max_len=3, eos_id=-7, n_draft=n_draft, temperature=temperature,
                                     generator=torch.Generator(device=DEV).manual_seed(5))
        one = G._PagedDecoder(m, nmr[:1], ir[:1], lambda P: P + 8, 8, 16)
        rows, last, c = torch.ones(N, dtype=torch.bool, device=DEV), 12, math.log(2 * 3 * V / 1e-9)
        for t in range(3):
            p = torch.softmax(one.step(torch.tensor([last], device=DEV)).double() / temperature, -1)[0].cpu()
            one.cache.lengths.add_(1)
            count = torch.bincount(got[rows, t + 1].cpu(), minlength=V).double()
            n = int(rows.sum())
            assert n >= 200
            assert ((count / n - p).abs() <= (2 * p * (1 - p) * c / n).sqrt() + 2 * c / (3 * n) + 1e-4).all(), t      # 1e-4: p in 32 bits
            last = int(count.argmax())
            rows &= got[:, t + 1] == last
    # each draft is checked against the very distribution that it was drawn from; no random number serves twice
    passes = len(calls) // T
    assert len(calls) == passes * T and passes >= 1
    for i in range(passes):
        *drawn, (drafts, p, u, q, _, accepted) = calls[i * T: (i + 1) * T]
        assert drafts.shape == (N, n_draft) and p.shape == (N, T, V) and q.shape == (N, n_draft, V)
        for j, (none, pj, _, qj, token, _) in enumerate(drawn):
            assert none.shape[1] == 0 and qj is None and torch.equal(pj[:, 0], q[:, j]) and torch.equal(token[:, 0], drafts[:, j])
    first = calls[n_draft][5].float().mean()
    assert 0.2 * n_draft < float(first) < 0.9 * n_draft or n_draft > 1               # drafts are neither all right nor all wrong
    u = torch.cat([x[2] for x in calls], 1)
    assert all(not torch.equal(u[:, i], u[:, j]) for i in range(u.shape[1]) for j in range(i))
