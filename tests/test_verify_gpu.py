"""ops.verify_drafts against its definition, evaluated in 64 bits on the host.  Outputs are whole numbers and have to be equal; the only
room is a random number within 2^-40 of a border, which the inputs here do not hit (checked)."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def _reference(x, p, u, q, counts):
    B, K = x.shape
    V = p.shape[2]
    tokens, accepted = np.full((B, K + 1), -1, dtype=np.int64), np.zeros(B, dtype=np.int32)
    for b in range(B):
        n = K if counts is None else min(max(int(counts[b]), 0), K)
        a = 0
        while a < n:
            t = int(x[b, a])
            if not 0 <= t < V:
                break
            if not u[b, a] * (1.0 if q is None else q[b, a, t]) < p[b, a, t]:
                break
            tokens[b, a] = t
            a += 1
        r = p[b, a].copy()
        if a < n:
            less = np.zeros(V)
            if q is not None:
                less = q[b, a]
            elif 0 <= int(x[b, a]) < V:
                less[int(x[b, a])] = 1.0
            rest = np.maximum(r - less, 0)
            r = rest if (rest > 0).any() else r
        c = np.cumsum(r)
        t = u[b, K] * c[-1]
        assert (np.abs(c - t)[r > 0] > 2.0 ** -40 * c[-1]).all() or t in (0.0,), "input on a border"
        over = np.flatnonzero(c > t)
        pos = np.flatnonzero(r > 0)
        tokens[b, a] = over[0] if len(over) else pos[-1] if len(pos) else 0
        accepted[b] = a
    return tokens, accepted


def _check(x, p, u, q=None, counts=None):
    from multimodal_amd import ops
    got, acc = ops.verify_drafts(x, p, u, q=q, counts=counts)
    h = lambda t: None if t is None else t.double().cpu().numpy() if t.is_floating_point() else t.cpu().numpy()
    want, wacc = _reference(h(x), h(p), h(u), h(q), h(counts))
    assert got.dtype == torch.int64 and acc.dtype == torch.int32
    assert (acc.cpu().numpy() == wacc).all()
    assert (got.cpu().numpy() == want).all(), np.argwhere(got.cpu().numpy() != want)[:5]
    return acc


def _inputs(seed, B, K, V, noise=0.7, scale=2.0):
    g = torch.Generator().manual_seed(seed)
    lp = torch.randn(B, K + 1, V, generator=g) * scale
    p = torch.softmax(lp, -1)
    q = torch.softmax(lp[:, :K] + noise * torch.randn(B, K, V, generator=g), -1)
    x = torch.multinomial(q.reshape(-1, V), 1, generator=g).view(B, K) if K else torch.zeros(B, 0, dtype=torch.long)
    return x.to(DEV), p.to(DEV), torch.rand(B, K + 1, generator=g).to(DEV), q.to(DEV), g


@pytest.mark.parametrize("with_q", [True, False])
@pytest.mark.parametrize("shape", [(1, 1, 2), (3, 0, 591), (16, 4, 591), (7, 5, 1), (5, 3, 1023), (4, 2, 4097), (2, 9, 50000), (3, 2, 128257), (300, 3, 77)],
                         ids=str)
def test_against_the_definition(shape, with_q):
    x, p, u, q, g = _inputs(1, *shape)
    _check(x, p, u, q if with_q else None)
    counts = torch.randint(-1, shape[1] + 2, (shape[0],), generator=g).int().to(DEV)
    _check(x, p, u, q if with_q else None, counts)


@pytest.mark.parametrize("with_q", [True, False])
@pytest.mark.parametrize("shape", [(130, 2, 50000), (128, 1, 12545), (1, 2, 1048577 + 300), (2, 1, 3000001)], ids=str)
def test_large_vocabularies(shape, with_q):
    """A workgroup a row with several blocks in flight (128 rows and more); blocks of more than 256 values (past 2^20), rows split over workgroups."""
    x, p, u, q, g = _inputs(11, *shape)
    _check(x, p, u, q if with_q else None)
    counts = torch.randint(0, shape[1] + 1, (shape[0],), generator=g).int().to(DEV)
    _check(x, p, u, q if with_q else None, counts)


def test_many_rows_of_a_vocabulary_past_2_to_the_20():
    """One distribution (batch stride 0), 200 random numbers: the place in its cumulative sum."""
    from multimodal_amd import ops
    V, B = 1048576 + 4099, 200
    g = torch.Generator().manual_seed(12)
    p = torch.softmax(torch.randn(V, generator=g) * 2, 0)
    u = torch.rand(B, 1, generator=g)
    c = p.double().numpy().cumsum()
    t = u[:, 0].double().numpy() * c[-1]
    want = np.searchsorted(c, t, side="right")
    assert (np.abs(c[want] - t) > 2.0 ** -40).all() and (np.abs(c[np.maximum(want - 1, 0)] - t) > 2.0 ** -40).all(), "input on a border"
    got, acc = ops.verify_drafts(torch.zeros(B, 0, dtype=torch.long, device=DEV), p.to(DEV).expand(B, 1, V), u.to(DEV))
    assert (got[:, 0].cpu().numpy() == want).all() and (acc == 0).all()


@pytest.mark.parametrize("B", [2, 130])
def test_empty_residuals_of_large_vocabularies(B):
    """p is half of q everywhere and the draft is rejected: nothing is left of p - q, so the last token is drawn from p itself.  Every third row's
    p is q: its draft is accepted."""
    _, p, u, q, g = _inputs(13, B, 1, 50000)
    p = torch.cat((q * 0.5, p[:, 1:]), 1)
    p[2::3, 0] = q[2::3, 0]
    x = torch.randint(0, 50000, (B, 1), generator=g).to(DEV)
    u[:, 0] = 0.5 + 0.25 * u[:, 0]
    acc = _check(x, p.contiguous(), u, q)
    assert acc.tolist() == [1 if b % 3 == 2 else 0 for b in range(B)]


def test_every_number_of_accepted_drafts_occurs():
    x, p, u, q, _ = _inputs(2, 400, 4, 50)
    acc = _check(x, p, u, q)
    assert set(acc.tolist()) == {0, 1, 2, 3, 4}


def test_strided_and_unaligned_rows():
    x, p, u, q, _ = _inputs(3, 6, 3, 1001)
    wide = torch.zeros(6, 5, 1010, device=DEV)
    wide[:, :4, 3:1004] = p
    qw = torch.zeros(6, 4, 1007, device=DEV)
    qw[:, :3, 1:1002] = q
    xs = torch.zeros(6, 8, dtype=torch.long, device=DEV); xs[:, 2:5] = x
    us = torch.zeros(6, 9, device=DEV); us[:, 1:5] = u
    _check(xs[:, 2:5], wide[:, :4, 3:1004], us[:, 1:5], qw[:, :3, 1:1002])
    _check(x, p[:1].expand(6, -1, -1), u, q[:1].expand(6, -1, -1))               # one distribution for all rows


def test_drafts_outside_the_vocabulary_and_empty_residuals():
    x, p, u, q, _ = _inputs(4, 8, 3, 100)
    x[0, 0], x[1, 1], x[2, 2] = -1, 100, 2 ** 40
    _check(x, p, u, q)
    _check(x, p, u)
    # p below q everywhere but at a draft that u = 1 - 2^-24 rejects: no residual, the row itself is drawn from
    p2 = torch.zeros(2, 2, 4, device=DEV); p2[:, :, 1] = 0.25; p2[:, :, 2] = 0.25; p2[1, 0, 3] = 0.5
    q2 = torch.zeros(2, 1, 4, device=DEV); q2[:, :, 1] = 0.5; q2[:, :, 2] = 0.5; q2[1, 0, 3] = 0.75
    x2 = torch.ones(2, 1, dtype=torch.long, device=DEV)
    acc = _check(x2, p2, torch.tensor([[1 - 2.0 ** -24, 0.7], [0.9, 0.3]], device=DEV), q2)
    assert acc.tolist() == [0, 0]
    # the target puts everything on the draft: a copied draft is accepted; a rejected one leaves nothing but the row
    one = torch.zeros(1, 2, 5, device=DEV); one[:, :, 3] = 1.0
    assert _check(torch.full((1, 1), 3, device=DEV), one, torch.tensor([[0.999, 0.5]], device=DEV)).tolist() == [1]
    assert _check(torch.full((1, 1), 2, device=DEV), one, torch.tensor([[0.0, 0.5]], device=DEV)).tolist() == [0]
    # no mass anywhere: token 0
    _check(torch.full((1, 1), 2, device=DEV), torch.zeros(1, 2, 5, device=DEV), torch.tensor([[0.5, 0.5]], device=DEV))


def test_extreme_random_numbers():
    """u = 0 takes the first token with any probability, u just below 1 the last; a sum that is not 1 scales along."""
    from multimodal_amd import ops
    for V in (10, 5000, 128257):
        p = torch.rand(4, 1, V, device=DEV) * 7
        p[:, :, :3] = 0
        p[:, :, -2:] = 0
        x = torch.zeros(4, 0, dtype=torch.long, device=DEV)
        first, _ = ops.verify_drafts(x, p, torch.zeros(4, 1, device=DEV))
        assert (first[:, 0] == (p[:, 0] > 0).long().argmax(-1)).all()
        tail, _ = ops.verify_drafts(x, p, torch.full((4, 1), 1 - 2.0 ** -24, device=DEV))
        c = p[:, 0].double().cumsum(-1)
        assert (tail[:, 0] == (c > (1 - 2.0 ** -24) * c[:, -1:]).long().argmax(-1)).all()
        beyond, _ = ops.verify_drafts(x, p, torch.full((4, 1), 1.0, device=DEV))      # outside [0, 1): the last token with any probability
        assert (beyond[:, 0] == V - 3).all()


def test_tokens_are_distributed_as_the_target():
    """Over a fine grid of (u_0, u_1) and a draft token drawn from q by a third grid, the first token's distribution is the target's."""
    from multimodal_amd import ops
    V, N = 6, 96
    g = torch.Generator().manual_seed(9)
    p0, q0 = torch.softmax(torch.randn(V, generator=g) * 1.5, 0), torch.softmax(torch.randn(V, generator=g), 0)
    grid = (torch.arange(N) + 0.5) / N
    u = torch.cartesian_prod(grid, grid)
    total = torch.zeros(V, dtype=torch.float64)
    for t in range(V):
        B = N * N
        p = p0.expand(B, 2, V).contiguous().to(DEV)
        toks, _ = ops.verify_drafts(torch.full((B, 1), t, device=DEV), p, u.float().to(DEV), q=q0.expand(B, 1, V).contiguous().to(DEV))
        total += q0[t].double() * torch.bincount(toks[:, 0].cpu(), minlength=V).double() / B
    # a probability measured on a grid of N points is off by at most 1/N per border: one border in u_0, two in u_1
    assert float((total - p0.double()).abs().max()) <= 3.0 / N


def test_captured_and_replayed_on_another_stream():
    from multimodal_amd import ops
    x, p, u, q, _ = _inputs(6, 9, 3, 3001)
    sets = [u, torch.rand_like(u), torch.rand_like(u)]
    want = [ops.verify_drafts(x, p, s, q=q) for s in sets]
    buf = u.clone()
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        g = torch.cuda.CUDAGraph()
        g.capture_begin()
        out = ops.verify_drafts(x, p, buf, q=q)
        g.capture_end()
    torch.cuda.synchronize()
    for w, n in zip(want, sets):
        buf.copy_(n)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], w[0]) and torch.equal(out[1], w[1])


def test_refusals():
    from multimodal_amd import ops
    x, p, u, q, _ = _inputs(7, 4, 3, 50)
    for change in (dict(drafts=x.int()), dict(drafts=x[0]), dict(drafts=x.cpu()), dict(p=p[:, :3]), dict(p=p.double()), dict(p=p.bfloat16()), dict(p=p.cpu()),
                   dict(u=u[:, :3]), dict(u=u.double()), dict(q=q[:, :2]), dict(q=q.double()), dict(counts=torch.ones(4, dtype=torch.long, device=DEV)),
                   dict(counts=torch.ones(3, dtype=torch.int32, device=DEV)), dict(p=p.transpose(1, 2)), dict(p=p[..., ::2]),
                   dict(p=p.clone().requires_grad_())):
        with pytest.raises((RuntimeError, TypeError)):
            ops.verify_drafts(**{**dict(drafts=x, p=p, u=u, q=q), **change})
    assert ops.verify_drafts(x[:0], p[:0], u[:0], q=q[:0])[0].shape == (0, 4)
