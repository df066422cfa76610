"""Paged key-value cache (ops.paged_cache_fill, paged_decode_attn, paged_evict) against its definition in 64 bits.

Tolerances, fixed before any run, for one output element of attention over n slots of a head of d:
  half a step of the output type (bf16 2^-8, f32 2^-24) times the value
  + E * sum_s p_s |v_s|, where E bounds the relative error of a probability and of the weighted sum:
      the score: d products and d sums in f32, (d + 8) 2^-24 of sum |q k| / sqrt(d) =: (d + 8) 2^-24 M; it enters p once directly and once
      through the normaliser;   exp / reciprocal and their arguments, 16 2^-24;   n + 8 roundings of each of the two sums;
      bf16: p is used as two bf16 terms, the first truncated (it leaves less than 2^-7 p, of which rounding the second loses 2^-8: 2^-15),
      and the rotated q as three truncated ones (8 bits each: 24, exact).
Stored keys: half a step of the type times the value + 4 2^-24 (|a| + |b|) of the pair that is rotated.  The attention reference
reads the keys as stored, which is what the operator is defined on.  Everything that is only moved is compared bit by bit."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
U = 2.0 ** -24


def _tables(rot, n):
    inv = 1.0 / (10000 ** (torch.arange(0, rot, 2, dtype=torch.float64) / max(rot, 1)))
    a = torch.arange(n, dtype=torch.float64)[:, None] * inv
    return a.cos().float().to(DEV), a.sin().float().to(DEV)


class Cache:
    """A pool with garbage (NaN) everywhere, pages dealt out at random, -1 in the table where a row has none."""

    def __init__(self, seed, dtype, B, Hkv, d, page, slots, spare=2, garbage=float("nan"), weights=False):
        g = torch.Generator().manual_seed(seed)
        need = [max(1, -(-max(s, 0) // page)) for s in slots]
        self.n_pages, self.page, self.dtype, self.Hkv, self.d = sum(need) + spare, page, dtype, Hkv, d
        perm = torch.randperm(self.n_pages, generator=g).tolist()
        table = torch.full((B, max(need)), -1, dtype=torch.int32)
        for b in range(B):
            for e in range(need[b]):
                table[b, e] = perm.pop()
        self.table = table.to(DEV)
        self.k = torch.full((self.n_pages, Hkv, page, d), garbage, dtype=dtype, device=DEV)
        self.v = torch.full_like(self.k, garbage)
        self.w = torch.full((self.n_pages, Hkv, page), garbage, device=DEV) if weights else None

    def rows(self, pool, b, n):
        """Slots 0 .. n-1 of row b: [Hkv, n, ...], float64 on the host."""
        pg = self.table[b].long().clamp(min=0)
        x = pool[pg].transpose(0, 1).flatten(1, 2)[:, :n]
        return x.double().cpu()

    def put(self, pool, b, n, values):
        """values [Hkv, n, ...] into slots 0 .. n-1 of row b (host loop over pages)."""
        for e in range(-(-n // self.page)):
            lo, hi = e * self.page, min(n, (e + 1) * self.page)
            pool[int(self.table[b, e]), :, : hi - lo] = values[:, lo:hi].to(pool.dtype).to(DEV)


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g).to(dtype)


def _turn(x, cos, sin, rot):
    """float64 half-layout rotation of x [..., d]; also the bound's |a| + |b|."""
    y, mag = x.clone(), torch.zeros_like(x)
    h = rot // 2
    if rot:
        a, b = x[..., :h], x[..., h:rot]
        y[..., :h], y[..., h:rot] = a * cos - b * sin, b * cos + a * sin
        mag[..., :h] = mag[..., h:rot] = a.abs() + b.abs()
    return y, mag


def _attend(q, K, V, there, stable, dtype):
    """q [H, d], K, V [Hkv, n, d], there [n]: (o [H, d], tolerance [H, d], p [H, n], relative error of p) in float64."""
    H, d = q.shape
    Hkv, n, _ = K.shape
    G = H // Hkv
    if not bool(there.any()):
        return torch.zeros(H, d, dtype=torch.float64), torch.zeros(H, d, dtype=torch.float64), torch.zeros(H, n, dtype=torch.float64), 0.0
    K, V = torch.where(there[:, None], K, torch.zeros(1, dtype=torch.float64)), torch.where(there[:, None], V, torch.zeros(1, dtype=torch.float64))
    K, V = K.repeat_interleave(G, 0), V.repeat_interleave(G, 0)
    x = (K * q[:, None]).sum(-1) / math.sqrt(d)
    M = float(((K * q[:, None]).abs().sum(-1) / math.sqrt(d)).max())
    if stable:
        p = torch.where(x < 0, 1 / (1 - x + 1e-9), x + 1) * there
        p = p / p.sum(-1, keepdim=True).clamp_min(1e-9)
    else:
        p = torch.softmax(x.masked_fill(~there, -math.inf), -1)
    o = (p[..., None] * V).sum(1)
    E = 2 * (d + 8) * U * M + 16 * U + 2 * (n + 8) * U
    tol = HALF[dtype] * o.abs() + (E + (2.0 ** -15 if dtype == torch.bfloat16 else 0.0)) * (1 + 2.0 ** -7) * (p[..., None] * V.abs()).sum(1)
    return o, tol, p, E + U


def _filled(seed, dtype, B, Hkv, G, d, page, lens, room=1, weights=False, spare=2):
    """A cache whose rows hold lens[b] random slots, and the inputs of one step (q, k, v slices of one fused row)."""
    g = torch.Generator().manual_seed(seed)
    c = Cache(seed, dtype, B, Hkv, d, page, [n + room for n in lens], weights=weights, spare=spare)
    for b, n in enumerate(lens):
        if n > 0:
            c.put(c.k, b, n, _randn(g, Hkv, n, d))
            c.put(c.v, b, n, _randn(g, Hkv, n, d))
            if weights:
                c.put(c.w, b, n, torch.rand(Hkv, n, generator=g))
    E = Hkv * d
    qkv = _randn(g, B, G * E + 2 * E + 4, dtype=dtype).to(DEV)
    return c, qkv[:, : G * E], qkv[:, G * E: G * E + E], qkv[:, G * E + E: G * E + 2 * E]


def _check_step(c, before, q, k, v, lens, H, rot, tabs, stable, positions, o, skip=()):
    """One step's outputs, stored slots, weights and everything it must leave alone.  before = (k, v, w) clones."""
    d, dtype = c.d, c.dtype
    bk, bv, bw = before
    hb, G = torch.arange(c.Hkv), H // c.Hkv
    wk, wv = bk.clone(), bv.clone()
    ww = None if bw is None else bw.clone()
    for b, n in enumerate(lens):
        o_b = o[b].double().cpu().view(H, d)
        if n < 0:
            assert (o_b == 0).all(), b
            continue
        at = n if k is not None else n - 1
        pos = min(max(int(positions[b]) if positions is not None else at, 0), (tabs[0].shape[0] if rot else 1) - 1)
        cs, sn = (t[pos].double().cpu() if rot else None for t in tabs)
        total = n
        if k is not None:
            total = n + 1
            e = n // c.page
            pg = int(c.table[b, e]) if e < c.table.shape[1] else -1
            if 0 <= pg < c.n_pages:
                want, mag = _turn(k[b].double().cpu().view(c.Hkv, d), cs, sn, rot)
                got = c.k[pg, :, n % c.page].double().cpu()
                assert ((got - want).abs() <= HALF[dtype] * want.abs() + 4 * U * mag).all(), ("stored key", b)
                assert torch.equal(c.v[pg, :, n % c.page], v[b].view(c.Hkv, d)), ("stored value", b)
                wk[pg, :, n % c.page] = c.k[pg, :, n % c.page]
                wv[pg, :, n % c.page] = c.v[pg, :, n % c.page]
                if ww is not None:
                    ww[pg, :, n % c.page] = 0
        total = min(total, c.table.shape[1] * c.page)
        pages = c.table[b].cpu()
        there = torch.tensor([0 <= int(pages[s // c.page]) < c.n_pages for s in range(total)], dtype=torch.bool)
        Q, _ = _turn(q[b].double().cpu().view(H, d), cs, sn, rot)
        valid = c.table[b].clamp(0, c.n_pages - 1).long()
        K = c.k[valid].transpose(0, 1).flatten(1, 2)[:, :total].double().cpu()
        V = c.v[valid].transpose(0, 1).flatten(1, 2)[:, :total].double().cpu()
        want, tol, p, E = _attend(Q, K, V, there, stable, dtype)
        assert torch.isfinite(o_b).all(), ("finite", b, n)
        bad = (o_b - want).abs() - tol
        assert (bad <= 0).all(), (b, n, float(bad.max()), float((o_b - want).abs().max()))
        if ww is not None:
            add = p.view(c.Hkv, G, total).sum(1)
            for s in range(total):
                if there[s]:
                    pg, off = int(pages[s // c.page]), s % c.page
                    w0 = ww[pg, :, off].double().cpu()
                    got = c.w[pg, :, off].double().cpu()
                    lim = (E + G * U) * add[:, s] + 2 * U * (w0.abs() + add[:, s])
                    assert ((got - w0 - add[:, s]).abs() <= lim).all(), ("weight", b, s, float((got - w0 - add[:, s]).abs().max()))
                    ww[pg, :, off] = c.w[pg, :, off]
    same = lambda a, b: torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))
    assert same(c.k, wk) and same(c.v, wv), "slots other than the appended ones were touched"
    if ww is not None:
        assert same(c.w, ww), "weights of slots that the rows do not hold were touched"


STEP = [
    # dtype, Hkv, G, d, page, lens, rot
    (torch.bfloat16, 1, 1, 128, 16, [0], 64),
    (torch.bfloat16, 8, 1, 128, 16, [170, 0, 1, 15, 16, 17, -1, 238], 64),
    (torch.float32, 8, 1, 128, 16, [170, 0, 1, 15, 16, 17, -1, 238], 64),
    (torch.bfloat16, 3, 1, 100, 4, [31, 32, 33, 3, 4], 50),
    (torch.float32, 3, 1, 100, 4, [31, 32, 33, 3, 4], 50),
    (torch.bfloat16, 2, 4, 64, 8, [1000, 7, 64, 63, 65], 64),
    (torch.float32, 2, 4, 64, 8, [1000, 7, 64, 63, 65], 0),
    (torch.bfloat16, 4, 2, 192, 32, [129, 511, 5], 96),
    (torch.float32, 4, 2, 192, 32, [129, 511, 5], 192),
    (torch.bfloat16, 1, 16, 256, 128, [700, 0], 0),
    (torch.bfloat16, 1, 20, 512, 64, [333, 2], 256),
    (torch.float32, 1, 20, 512, 64, [333, 2], 256),
    (torch.bfloat16, 2, 5, 4, 16, [40, 3], 4),
    (torch.float32, 2, 33, 36, 1024, [1100], 18),
    (torch.bfloat16, 2, 3, 260, 16, [75, 20], 130),
    (torch.bfloat16, 5, 7, 96, 16, [2500, 1, 300], 96),
]


@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("stable", [False, True])
@pytest.mark.parametrize("case", STEP, ids=lambda c: f"{str(c[0])[6:]}-Hkv{c[1]}xG{c[2]}-d{c[3]}-page{c[4]}-rot{c[6]}")
def test_step_against_the_definition(case, stable, weights):
    from multimodal_amd import ops
    dtype, Hkv, G, d, page, lens, rot = case
    c, q, k, v = _filled(3, dtype, len(lens), Hkv, G, d, page, lens, weights=weights)
    before = (c.k.clone(), c.v.clone(), None if c.w is None else c.w.clone())
    tabs = _tables(rot, max(lens) + 1)
    n = torch.tensor(lens, dtype=torch.int32, device=DEV)
    o = ops.paged_decode_attn(q, k, v, c.k, c.v, c.table, n, Hkv * G, rot, *tabs, stable, weights=c.w)
    assert torch.equal(n.cpu(), torch.tensor(lens, dtype=torch.int32))
    _check_step(c, before, q, k, v, lens, Hkv * G, rot, tabs, stable, None, o)
    # the same step again, on what it has stored: the same bits
    if not weights:
        assert torch.equal(o, ops.paged_decode_attn(q, k, v, c.k, c.v, c.table, n, Hkv * G, rot, *tabs, stable))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_step_without_a_new_token(dtype):
    """k_new = None: only what is stored; a row without a slot gets zeros, the rotary position defaults to the last slot."""
    from multimodal_amd import ops
    lens = [0, 1, 77, -1, 200]
    c, q, _, _ = _filled(5, dtype, 5, 2, 3, 64, 16, lens, weights=True)
    before = (c.k.clone(), c.v.clone(), c.w.clone())
    tabs = _tables(32, 201)
    o = ops.paged_decode_attn(q, None, None, c.k, c.v, c.table, torch.tensor(lens, dtype=torch.int32, device=DEV), 6, 32, *tabs, False, weights=c.w)
    _check_step(c, before, q, None, None, lens, 6, 32, tabs, False, None, o)
    assert (o[0] == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rotary_positions_apart_from_the_slots(dtype):
    """positions: after an eviction the slot says nothing about the position; values past the tables are clamped to them."""
    from multimodal_amd import ops
    lens, pos = [10, 20, 30, 0], [500, 3, 100000, -7]
    c, q, k, v = _filled(6, dtype, 4, 2, 2, 64, 8, lens)
    before = (c.k.clone(), c.v.clone(), None)
    tabs = _tables(64, 600)
    o = ops.paged_decode_attn(q, k, v, c.k, c.v, c.table, torch.tensor(lens, dtype=torch.int32, device=DEV), 4, 64, *tabs, False,
                              positions=torch.tensor(pos, dtype=torch.int32, device=DEV))
    _check_step(c, before, q, k, v, lens, 4, 64, tabs, False, pos, o)


@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_pages_the_table_does_not_hold(dtype, weights):
    """Page numbers outside the pool, in the middle of a row, at its end and for the new token, and rows longer than their table: those slots
    are neither read nor written."""
    from multimodal_amd import ops
    lens = [100, 64, 200, 37, 128, 31]
    c, q, k, v = _filled(7, dtype, 6, 2, 2, 64, 16, lens, weights=weights)
    c.table[0, 2] = -1                                   # a hole
    c.table[1, 4] = c.n_pages                            # the new token's page
    c.table[2, 1] = 2 ** 31 - 1
    c.table[2, 12] = -2 ** 31                            # the last page, new token's among its slots
    c.table[3] = -5                                      # nothing at all
    c.table = c.table[:, :8].contiguous()                # rows 2 and 4 are longer than this: row 4's new token has no page
    before = (c.k.clone(), c.v.clone(), None if c.w is None else c.w.clone())
    tabs = _tables(64, 256)
    o = ops.paged_decode_attn(q, k, v, c.k, c.v, c.table, torch.tensor(lens, dtype=torch.int32, device=DEV), 4, 64, *tabs, False, weights=c.w)
    _check_step(c, before, q, k, v, lens, 4, 64, tabs, False, None, o)
    assert (o[3] == 0).all()


def test_non_finite_slots_that_count_and_that_do_not():
    """A NaN key inside the row reaches only its row; an infinite value its column; NaN behind the row or in free pages nothing."""
    from multimodal_amd import ops
    for dtype in (torch.bfloat16, torch.float32):
        lens = [50, 50, 50]
        c, q, k, v = _filled(8, dtype, 3, 1, 2, 64, 16, lens)
        c.k[int(c.table[1, 1]), 0, 5, 7] = float("nan")
        c.v[int(c.table[2, 2]), 0, 3, 9] = float("inf")
        o = ops.paged_decode_attn(q, k, v, c.k, c.v, c.table, torch.tensor(lens, dtype=torch.int32, device=DEV), 2, 0, None, None, False).float()
        assert torch.isfinite(o[0]).all() and torch.isnan(o[1]).all()
        o2 = o[2].view(2, 64)
        assert torch.isinf(o2[:, 9]).all() and torch.isfinite(torch.cat((o2[:, :9], o2[:, 10:]), 1)).all()


def test_an_infinite_key_weighs_nothing_or_everything():
    """A key with -inf where q is positive scores -inf: weight 0, the row as without it (rotated q: three terms, none of them 0)."""
    from multimodal_amd import ops
    for dtype in (torch.bfloat16, torch.float32):
        c, q, k, v = _filled(18, dtype, 1, 1, 1, 64, 16, [50])
        n = torch.tensor([50], dtype=torch.int32, device=DEV)
        q = q.abs().clone()
        q[0, 40] = 1.5                                                                    # exact in one term
        tabs = _tables(64, 51)
        tabs = (tabs[0].clone().fill_(1.0), tabs[1].clone().fill_(0.0))                   # a rotation by nothing
        for col in (40, 7):
            c.k[int(c.table[0, 1]), 0, 5] = 0
            c.k[int(c.table[0, 1]), 0, 5, col] = -math.inf
            o = ops.paged_decode_attn(q, k, v, c.k, c.v, c.table, n, 1, 64, *tabs, False)
            K, V = c.rows(c.k, 0, 51), c.rows(c.v, 0, 51)
            keep = torch.arange(51) != 21
            want, tol, _, _ = _attend(q[0].double().cpu().view(1, 64), K[:, keep], V[:, keep], torch.ones(50, dtype=torch.bool), False, dtype)
            assert ((o.double().cpu().view(1, 64) - want).abs() <= tol).all()


def test_an_infinite_query_weighs_its_keys_by_sign():
    """A rotated query with an infinite pair: keys that are negative there score -inf.  Where all are, the row is without weight; where the others
    are 0 there, or positive, there is no finite answer."""
    from multimodal_amd import ops
    for dtype in (torch.bfloat16, torch.float32):
        for stable in (False, True):
            c, q, k, v = _filled(25, dtype, 2, 1, 2, 64, 16, [50, 50])
            q = q.clone()
            q[:, 7], q[:, 39] = math.inf, 1.0                                             # the pair (7, 39) of head 0; head 1 is finite
            c.k[..., 7], c.k[..., 39] = -0.5, -0.25
            c.k[int(c.table[1, 1]), 0, 3, 7] = 0.5
            c.k[int(c.table[1, 1]), 0, 3, 39] = 0.5
            tabs = tuple(torch.full((50, 32), x, device=DEV) for x in (0.8, 0.6))         # both of the pair become +inf
            n = torch.tensor([50, 50], dtype=torch.int32, device=DEV)
            o = ops.paged_decode_attn(q, None, None, c.k, c.v, c.table, n, 2, 64, *tabs, stable).float().view(2, 2, 64)
            assert (o[0, 0] == 0).all() and torch.isnan(o[1, 0]).all() and torch.isfinite(o[:, 1]).all(), (dtype, stable)


def test_large_scores_do_not_overflow():
    """Scores far beyond exp's range, of both signs: the running maximum keeps the sums finite."""
    from multimodal_amd import ops
    for dtype in (torch.bfloat16, torch.float32):
        lens = [300, 90]
        c, q, k, v = _filled(9, dtype, 2, 2, 2, 64, 16, lens)
        q = (q * 40).to(dtype)
        before = (c.k.clone(), c.v.clone(), None)
        o = ops.paged_decode_attn(q, k, v, c.k, c.v, c.table, torch.tensor(lens, dtype=torch.int32, device=DEV), 4, 0, None, None, False)
        _check_step(c, before, q, k, v, lens, 4, 0, (None, None), False, None, o)


@pytest.mark.parametrize("stable", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_large_values_count_by_their_weight_alone(dtype, stable):
    """Values of 2^100 in slots whose probability is nothing (softmax, 200 and more below the maximum: exp underflows) or about 2^-117
    (stablemax's s(x) = 1 / (1 - x) far down): the sum gets p v of them and no more.  Each p may be off by 2^-126, the least normal number, on
    top of the bound above, whose M is that of the ordinary slots: the others' p is relative to their score in stablemax, 0 in softmax."""
    from multimodal_amd import ops
    lens, H, d = [200, 1500], 2, 64
    c, q, k, v = _filled(21, dtype, 2, 1, H, d, 16, lens)
    q = (q.abs() + 0.5).to(dtype)
    for b, n in enumerate(lens):
        s = torch.arange(1, n, 3)
        pg, off = c.table[b].cpu().long()[s // 16].to(DEV), (s % 16).to(DEV)
        c.k[pg, :, off] = -(2.0 ** 112) if stable else -60.0
        c.v[pg, :, off] = 2.0 ** 100
    n_dev = torch.tensor(lens, dtype=torch.int32, device=DEV)
    o = ops.paged_decode_attn(q, None, None, c.k, c.v, c.table, n_dev, H, 0, None, None, stable).double().cpu()
    for b, n in enumerate(lens):
        Q, K, V = q[b].double().cpu().view(H, d), c.rows(c.k, b, n), c.rows(c.v, b, n)
        there = torch.ones(n, dtype=torch.bool)
        ordinary = there.clone(); ordinary[1::3] = False
        want, _, p, _ = _attend(Q, K, V, there, stable, dtype)
        E = _attend(Q, K, V, ordinary, stable, dtype)[3]
        tol = HALF[dtype] * want.abs() + (E + (2.0 ** -15 if dtype == torch.bfloat16 else 0.0)) * (1 + 2.0 ** -7) * (p[..., None] * V.abs()).sum(1) \
            + n * 2.0 ** -126 * 2.0 ** 100
        assert ((o[b].view(H, d) - want).abs() <= tol).all(), (b, float((o[b].view(H, d) - want).abs().max()))


def test_small_queries_of_large_keys():
    """Rotated queries near 2^-100 of keys near 2^100: the scores are ordinary ones.  A term of q may be off by 2^-126, two of them a value."""
    from multimodal_amd import ops
    for dtype in (torch.bfloat16, torch.float32):
        n, H, d = 90, 2, 64
        c, q, _, _ = _filled(23, dtype, 1, 1, H, d, 16, [n])
        q, c.k = (q.float() * 2.0 ** -100).to(dtype), (c.k.float() * 2.0 ** 100).to(dtype)
        tabs = _tables(64, n)
        o = ops.paged_decode_attn(q, None, None, c.k, c.v, c.table, torch.tensor([n], dtype=torch.int32, device=DEV), H, 64, *tabs, False).double().cpu()
        Q, _ = _turn(q[0].double().cpu().view(H, d), tabs[0][n - 1].double().cpu(), tabs[1][n - 1].double().cpu(), 64)
        K, V = c.rows(c.k, 0, n), c.rows(c.v, 0, n)
        want, tol, p, _ = _attend(Q, K, V, torch.ones(n, dtype=torch.bool), False, dtype)
        turned = 4 * U * float((K.abs() * 1.5 * Q.abs().max()).sum(-1).max()) / math.sqrt(d)          # rounding of the rotated q: as of stored keys
        floor = 2 * 2.0 ** -126 * float(K.abs().sum(-1).max()) / math.sqrt(d)
        assert ((o.view(H, d) - want).abs() <= tol + 2 * (turned + floor) * (p[..., None] * V.abs()).sum(1)).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_long_rows_beside_short_ones(dtype):
    """Lengths far apart in one call (the cache's length is split over workgroups), with weights."""
    from multimodal_amd import ops
    lens = [9001, 1, 4096, 0, 4095, 255, 256, 257]
    c, q, k, v = _filled(10, dtype, len(lens), 1, 2, 64, 64, lens, weights=True)
    before = (c.k.clone(), c.v.clone(), c.w.clone())
    tabs = _tables(64, 9002)
    o = ops.paged_decode_attn(q, k, v, c.k, c.v, c.table, torch.tensor(lens, dtype=torch.int32, device=DEV), 2, 64, *tabs, False, weights=c.w)
    _check_step(c, before, q, k, v, lens, 2, 64, tabs, False, None, o)


@pytest.mark.parametrize("dtype,G,d,width,weights", [
    (torch.bfloat16, 1, 64, 0, False), (torch.bfloat16, 4, 36, 0, True), (torch.float32, 2, 64, 0, False), (torch.bfloat16, 3, 128, 32, False),
    (torch.float32, 1, 100, 32, True), (torch.bfloat16, 8, 64, 32, False), (torch.bfloat16, 1, 512, 32, False), (torch.float32, 1, 512, 32, False)])
def test_many_short_rows(dtype, G, d, width, weights):
    """More rows and heads than the card has waves, of 0 to 60 slots: a wave each (up to four query heads a KV head).  width = 32: tables as wide
    as 512 slots, a cache too large for the last-level cache by what it could hold.  A few rows against the definition, all of them against
    a call of their own."""
    from multimodal_amd import ops
    B, Hkv, rot = 512, 4, d // 4 * 2
    g = torch.Generator().manual_seed(14)
    lens = torch.randint(-1, 61, (B,), generator=g).tolist()
    c, q, k, v = _filled(14, dtype, B, Hkv, G, d, 16, lens, weights=weights)
    if width:
        c.table = torch.nn.functional.pad(c.table, (0, width - c.table.shape[1]), value=-1).contiguous()
    before = (c.k.clone(), c.v.clone(), None if c.w is None else c.w.clone())
    tabs = _tables(rot, 61)
    n = torch.tensor(lens, dtype=torch.int32, device=DEV)
    o = ops.paged_decode_attn(q, k, v, c.k, c.v, c.table, n, Hkv * G, rot, *tabs, False, weights=c.w)
    few = list(range(0, B, 37))
    sub = Cache.__new__(Cache)
    sub.__dict__.update(c.__dict__)
    sub.table = c.table[few].contiguous()
    # what the other rows did to their own pages is theirs: the check of untouched slots takes it as given
    mine = torch.zeros(c.n_pages, dtype=torch.bool, device=DEV)
    mine[sub.table[sub.table >= 0].long()] = True
    base = tuple(None if x is None else torch.where(mine.view(-1, *[1] * (x.dim() - 1)), x, y) for x, y in zip(before, (c.k, c.v, c.w)))
    _check_step(sub, base, q[few], k[few], v[few], [lens[b] for b in few], Hkv * G, rot, tabs, False, None, o[few])
    for i in range(0, B, 64):
        s = slice(i, i + 64)
        part = ops.paged_decode_attn(q[s], None, None, c.k, c.v, c.table[s], torch.where(n[s] < 0, n[s], n[s] + 1), Hkv * G, rot, *tabs, False)
        # two evaluations of the same stored slots: each within the bound, whose sum part is below 2^-12 of the largest value here
        assert ((part.float() - o[s].float()).abs() <= 2 * HALF[dtype] * o[s].float().abs() + 2.0 ** -12 * float(o.float().abs().max())).all(), i


@pytest.mark.parametrize("dtype,G,d", [(torch.bfloat16, 3, 128), (torch.float32, 1, 100), (torch.bfloat16, 8, 72), (torch.bfloat16, 1, 512), (torch.float32, 1, 512),
                                       (torch.bfloat16, 5, 100), (torch.float32, 5, 200)])
def test_pools_past_the_last_level_cache(dtype, G, d):
    """Pools of more than 256 MB that the tables can name whole (read non-temporally), a wave a row and four: a few rows against the definition,
    all of them against calls of a few rows, which read through the caches."""
    from multimodal_amd import ops
    B, Hkv, rot, width = 640, 4, d // 4 * 2, 32
    g = torch.Generator().manual_seed(24)
    lens = torch.randint(-1, 61, (B,), generator=g).tolist()
    c, q, k, v = _filled(24, dtype, B, Hkv, G, d, 16, lens, spare=(256 << 20) // (16 * Hkv * d * 2 * dtype.itemsize) + 1)
    c.table = torch.nn.functional.pad(c.table, (0, width - c.table.shape[1]), value=-1).contiguous()
    assert min(c.n_pages, B * width) * 16 * Hkv * d * 2 * dtype.itemsize > 256 << 20
    before = (c.k.clone(), c.v.clone(), None)
    tabs = _tables(rot, 61)
    n = torch.tensor(lens, dtype=torch.int32, device=DEV)
    o = ops.paged_decode_attn(q, k, v, c.k, c.v, c.table, n, Hkv * G, rot, *tabs, False)
    few = list(range(0, B, 53))
    sub = Cache.__new__(Cache)
    sub.__dict__.update(c.__dict__)
    sub.table = c.table[few].contiguous()
    mine = torch.zeros(c.n_pages, dtype=torch.bool, device=DEV)
    mine[sub.table[sub.table >= 0].long()] = True
    base = tuple(torch.where(mine.view(-1, 1, 1, 1), x, y) for x, y in zip(before, (c.k, c.v))) + (None,)
    _check_step(sub, base, q[few], k[few], v[few], [lens[b] for b in few], Hkv * G, rot, tabs, False, None, o[few])
    del before, base
    for i in range(0, B, 64):
        s = slice(i, i + 64)
        part = ops.paged_decode_attn(q[s], None, None, c.k, c.v, c.table[s], torch.where(n[s] < 0, n[s], n[s] + 1), Hkv * G, rot, *tabs, False)
        # as in test_many_short_rows
        assert ((part.float() - o[s].float()).abs() <= 2 * HALF[dtype] * o[s].float().abs() + 2.0 ** -12 * float(o.float().abs().max())).all(), i


def test_tables_far_wider_than_the_rows():
    """A table of 200000 slots for rows of a few: splits beyond a row's end do nothing."""
    from multimodal_amd import ops
    for dtype in (torch.bfloat16, torch.float32):
        lens = [700, 3, 0, -1]
        c, q, k, v = _filled(15, dtype, 4, 2, 2, 64, 32, lens, weights=True)
        c.table = torch.nn.functional.pad(c.table, (0, 6250 - c.table.shape[1]), value=-1).contiguous()
        before = (c.k.clone(), c.v.clone(), c.w.clone())
        n = torch.tensor(lens, dtype=torch.int32, device=DEV)
        o = ops.paged_decode_attn(q, k, v, c.k, c.v, c.table, n, 4, 0, None, None, False, weights=c.w)
        c.table = c.table[:, :40].contiguous()
        _check_step(c, before, q, k, v, lens, 4, 0, (None, None), False, None, o)


def test_offsets_past_32_bits():
    """A pool of more than 2^32 bytes and 2^31 elements: pages at its end (store, attend, fill, evict)."""
    from multimodal_amd import ops
    page, d, Hkv = 1024, 128, 4
    n_pages = (1 << 31) // (page * d * Hkv) + 9
    c = Cache(1, torch.bfloat16, 1, Hkv, d, page, [1], spare=0)
    c.n_pages = n_pages
    c.k = torch.zeros(n_pages, Hkv, page, d, dtype=torch.bfloat16, device=DEV)
    c.v = torch.zeros_like(c.k)
    c.w = torch.zeros(n_pages, Hkv, page, device=DEV)
    c.table = torch.tensor([[n_pages - 1, n_pages - 3]], dtype=torch.int32, device=DEV)
    g = torch.Generator().manual_seed(2)
    kv = _randn(g, 1, 1100, 2 * Hkv * d, dtype=torch.bfloat16).to(DEV)
    ops.paged_cache_fill(kv[:, :, : Hkv * d], kv[:, :, Hkv * d:], c.k, c.v, c.table, 0, None, None, weights=c.w)
    flat = kv[0].view(1100, 2, Hkv, d)
    assert torch.equal(c.k[n_pages - 1], flat[:1024, 0].transpose(0, 1)) and torch.equal(c.v[n_pages - 3, :, :76], flat[1024:, 1].transpose(0, 1))
    q = _randn(g, 1, 3 * Hkv * d, dtype=torch.bfloat16).to(DEV)
    n = torch.tensor([1100], dtype=torch.int32, device=DEV)
    o = ops.paged_decode_attn(q[:, : Hkv * d], q[:, Hkv * d: 2 * Hkv * d], q[:, 2 * Hkv * d:], c.k, c.v, c.table, n, Hkv, 0, None, None, False,
                              weights=c.w)
    K = c.k[c.table[0].long()].transpose(0, 1).flatten(1, 2)[:, :1101].double().cpu()
    V = c.v[c.table[0].long()].transpose(0, 1).flatten(1, 2)[:, :1101].double().cpu()
    want, tol, p, E = _attend(q[0, : Hkv * d].double().cpu().view(Hkv, d), K, V, torch.ones(1101, dtype=torch.bool), False, torch.bfloat16)
    assert ((o.double().cpu().view(Hkv, d) - want).abs() <= tol).all()
    got = c.w[c.table[0].long()].transpose(0, 1).flatten(1, 2)[:, :1101].double().cpu()
    assert ((got - p).abs() <= (E + 4 * U) * p).all()
    n.fill_(1101)
    kept = ops.paged_evict(c.k, c.v, c.w, c.table, n, 1050, 40)
    moved = kept[0].long().cpu()
    got = c.k[c.table[0].long()].transpose(0, 1).flatten(1, 2)[:, :1050].double().cpu()
    assert torch.equal(got, torch.stack([K[h, moved[h]] for h in range(Hkv)]))
    assert int((c.k[: n_pages - 3] != 0).sum()) == 0 and int((c.v[: n_pages - 3] != 0).sum()) == 0


def test_shared_prompt_pages_and_repeated_rows():
    """Rows whose tables share read-only pages, and a table row repeated for several queries (stride 0 as well)."""
    from multimodal_amd import ops
    c, q, k, v = _filled(11, torch.bfloat16, 3, 2, 1, 64, 16, [64, 64, 64])
    c.table[1, :4] = c.table[0, :4]
    c.table[2, :4] = c.table[0, :4]
    n = torch.tensor([64, 64, 64], dtype=torch.int32, device=DEV)
    o = ops.paged_decode_attn(q, k, v, c.k, c.v, c.table, n, 2, 0, None, None, False)
    for b in range(3):
        o1 = ops.paged_decode_attn(q[b:b + 1], k[b:b + 1], v[b:b + 1], c.k, c.v, c.table[b:b + 1], n[b:b + 1], 2, 0, None, None, False)
        assert torch.equal(o1, o[b:b + 1])
    oe = ops.paged_decode_attn(q, None, None, c.k, c.v, c.table[:1].expand(3, -1), n, 2, 0, None, None, False)
    for b in range(3):
        assert torch.equal(oe[b:b + 1], ops.paged_decode_attn(q[b:b + 1], None, None, c.k, c.v, c.table[:1], n[:1], 2, 0, None, None, False))


@pytest.mark.parametrize("dtype,d,rot", [(torch.bfloat16, 64, 64), (torch.bfloat16, 100, 50), (torch.float32, 64, 32), (torch.float32, 36, 6)])
def test_rows_at_odd_addresses(dtype, d, rot):
    """q, k and v as views whose rows start at any multiple of a value's size: the step and the run."""
    from multimodal_amd import ops
    lens = [40, 0, 17]
    Hkv, G = 2, 3
    c, q, k, v = _filled(16, dtype, 3, Hkv, G, d, 16, lens, weights=True)
    g = torch.Generator().manual_seed(17)
    odd = lambda *s: _randn(g, *s[:-1], s[-1] + 7, dtype=dtype).to(DEV)[..., 3: 3 + s[-1]]
    q, k, v = odd(3, Hkv * G * d), odd(3, Hkv * d), odd(3, Hkv * d)
    assert q.data_ptr() % 4 == (2 if dtype == torch.bfloat16 else 0)
    before = (c.k.clone(), c.v.clone(), c.w.clone())
    tabs = _tables(rot, 50)
    n = torch.tensor(lens, dtype=torch.int32, device=DEV)
    o = ops.paged_decode_attn(q, k, v, c.k, c.v, c.table, n, Hkv * G, rot, *tabs, False, weights=c.w)
    _check_step(c, before, q, k, v, lens, Hkv * G, rot, tabs, False, None, o)
    kk, vv = odd(3, 4, Hkv * d), odd(3, 4, Hkv * d)
    a, b = Cache(19, dtype, 3, Hkv, d, 16, [60] * 3), Cache(19, dtype, 3, Hkv, d, 16, [60] * 3)
    ops.paged_cache_fill(kk, vv, a.k, a.v, a.table, rot, *tabs, start=n)
    ops.paged_cache_fill(kk.contiguous(), vv.contiguous(), b.k, b.v, b.table, rot, *tabs, start=n)
    assert torch.equal(a.k.view(torch.uint8), b.k.view(torch.uint8)) and torch.equal(a.v.view(torch.uint8), b.v.view(torch.uint8))


def test_all_scores_minus_infinity():
    """Every key infinitely far away: a row without weight gets zeros."""
    from multimodal_amd import ops
    for dtype in (torch.bfloat16, torch.float32):
        c, q, k, v = _filled(20, dtype, 1, 1, 1, 64, 16, [40])
        q = q.clone().fill_(1.0)
        c.k[c.table[0].long()] = -math.inf
        o = ops.paged_decode_attn(q, None, None, c.k, c.v, c.table, torch.tensor([40], dtype=torch.int32, device=DEV), 1, 0, None, None, False)
        assert (o == 0).all()


def test_agrees_with_the_dense_cache_step():
    """The same step through ops.decode_attn's dense cache: float32, both normalisations."""
    from multimodal_amd import ops
    B, H, d, n, rot = 4, 4, 128, 57, 64
    c, q, k, v = _filled(12, torch.float32, B, H, 1, d, 16, [n] * B)
    kc = torch.zeros(B, H, 64, d, device=DEV); vc = torch.zeros_like(kc)
    for b in range(B):
        kc[b, :, :n] = c.rows(c.k, b, n).float().to(DEV); vc[b, :, :n] = c.rows(c.v, b, n).float().to(DEV)
    tabs = _tables(rot, 64)
    fused = torch.cat((q, k, v), 1)
    E = H * d
    for stable in (False, True):
        want = ops.decode_attn(fused[:, :E], fused[:, E:2 * E], fused[:, 2 * E:], kc, vc, H, rot, n, *tabs, stable)
        got = ops.paged_decode_attn(fused[:, :E], fused[:, E:2 * E], fused[:, 2 * E:], c.k, c.v, c.table,
                                    torch.full((B,), n, dtype=torch.int32, device=DEV), H, rot, *tabs, stable)
        # two float32 evaluations, each within E of the definition: E * max|v| with M <= 2 |q||k| / sqrt(d) < 40 here
        assert float((got - want).abs().max()) <= 2 * (2 * (d + 8) * U * 40 + 16 * U + 2 * (n + 9) * U) * float(vc.abs().max())


# ------------------------------------------------------------------------------------------------ runs
FILL = [
    # dtype, B, Hkv, d, page, S, rot, start, counts, positions
    (torch.bfloat16, 3, 8, 128, 16, 40, 64, None, [40, 7, 0], None),
    (torch.float32, 3, 2, 100, 4, 33, 50, [0, 5, 61], [33, 1, 20], None),
    (torch.bfloat16, 2, 3, 100, 8, 21, 50, [3, 0], None, [700, 5]),
    (torch.bfloat16, 4, 2, 64, 32, 1, 64, [0, 31, 32, -1], None, None),
    (torch.float32, 2, 1, 4, 1024, 5, 2, None, [100, -3], None),
    (torch.bfloat16, 2, 2, 512, 16, 19, 256, [15, 16], None, None),
    (torch.bfloat16, 2, 2, 72, 16, 19, 34, [15, 16], None, None),
    (torch.float32, 1, 5, 64, 16, 130, 0, None, None, None),
]


@pytest.mark.parametrize("case", FILL, ids=lambda c: f"{str(c[0])[6:]}-B{c[1]}-d{c[3]}-page{c[4]}-S{c[5]}-rot{c[6]}")
def test_fill_against_the_definition(case):
    from multimodal_amd import ops
    dtype, B, Hkv, d, page, S, rot, start, counts, positions = case
    g = torch.Generator().manual_seed(21)
    st = start or [0] * B
    n = [min(x, S) for x in (counts or [S] * B)]
    c = Cache(21, dtype, B, Hkv, d, page, [max(a, 0) + b for a, b in zip(st, n)], weights=True)
    tabs = _tables(rot, 800)
    E = Hkv * d
    kv = torch.full((B, S + 2, 2 * E + 8), float("nan"), dtype=dtype)                    # a padded batch: what counts leave out is garbage
    for b in range(B):
        kv[b, : max(n[b], 0)] = _randn(g, max(n[b], 0), 2 * E + 8, dtype=dtype)
    kv = kv.to(DEV)
    k, v = kv[:, :S, :E], kv[:, :S, E + 8: 2 * E + 8]
    before = (c.k.clone(), c.v.clone(), c.w.clone())
    i32 = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32, device=DEV)
    ops.paged_cache_fill(k, v, c.k, c.v, c.table, rot, *tabs, start=i32(start), counts=i32(counts), positions=i32(positions), weights=c.w)
    wk, wv, ww = before
    for b in range(B):
        if st[b] < 0:
            continue
        for s in range(n[b]):
            slot = st[b] + s
            pg, off = int(c.table[b, slot // page]), slot % page
            pos = (positions[b] if positions else st[b]) + s
            want, mag = _turn(k[b, s].double().cpu().view(Hkv, d), tabs[0][pos].double().cpu(), tabs[1][pos].double().cpu(), rot)
            got = c.k[pg, :, off].double().cpu()
            assert ((got - want).abs() <= HALF[dtype] * want.abs() + 4 * U * mag).all(), (b, s)
            assert torch.equal(c.v[pg, :, off], v[b, s].view(Hkv, d))
            wk[pg, :, off], wv[pg, :, off], ww[pg, :, off] = c.k[pg, :, off], c.v[pg, :, off], 0
    same = lambda a, b: torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))
    assert same(c.k, wk) and same(c.v, wv) and same(c.w, ww)


def test_fill_leaves_out_pages_the_table_does_not_hold():
    from multimodal_amd import ops
    c = Cache(22, torch.bfloat16, 2, 2, 64, 16, [64, 64])
    c.table[0, 1] = -1
    c.table[1, 3] = c.n_pages
    before = (c.k.clone(), c.v.clone())
    kv = torch.randn(2, 100, 256, device=DEV).bfloat16()                                 # 100 tokens for rows of 64 slots
    ops.paged_cache_fill(kv[..., :128], kv[..., 128:], c.k, c.v, c.table, 0, None, None)
    wk, wv = before
    for b, bad in ((0, 1), (1, 3)):
        for e in range(4):
            if e != bad:
                pg = int(c.table[b, e])
                wk[pg] = kv[b, e * 16: e * 16 + 16, :128].view(16, 2, 64).transpose(0, 1)
                wv[pg] = kv[b, e * 16: e * 16 + 16, 128:].view(16, 2, 64).transpose(0, 1)
    same = lambda a, b: torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    assert same(c.k, wk) and same(c.v, wv)


def test_drafted_tokens_in_one_call_equal_one_by_one():
    """paged_cache_fill of T tokens and one attention row per token (its table row repeated, its own length) against T appending steps:
    the keys are the same bits; the outputs too, as both attend over the same stored slots."""
    from multimodal_amd import ops
    for dtype in (torch.bfloat16, torch.float32):
        lens, T, Hkv, G, d, rot = [37, 0, 90], 5, 2, 2, 64, 32
        g = torch.Generator().manual_seed(30)
        a, _, _, _ = _filled(30, dtype, 3, Hkv, G, d, 16, lens, room=T)
        b, _, _, _ = _filled(30, dtype, 3, Hkv, G, d, 16, lens, room=T)
        tabs = _tables(rot, 128)
        q = _randn(g, 3, T, Hkv * G * d, dtype=dtype).to(DEV)
        k, v = _randn(g, 3, T, Hkv * d, dtype=dtype).to(DEV), _randn(g, 3, T, Hkv * d, dtype=dtype).to(DEV)
        n = torch.tensor(lens, dtype=torch.int32, device=DEV)
        ops.paged_cache_fill(k, v, a.k, a.v, a.table, rot, *tabs, start=n)
        rows = (n[:, None] + torch.arange(1, T + 1, dtype=torch.int32, device=DEV)).reshape(-1)
        many = ops.paged_decode_attn(q.view(3 * T, -1), None, None, a.k, a.v, a.table.repeat_interleave(T, 0), rows, Hkv * G, rot, *tabs, False)
        for t in range(T):
            one = ops.paged_decode_attn(q[:, t], k[:, t], v[:, t], b.k, b.v, b.table, n + t, Hkv * G, rot, *tabs, False)
            tol = 4 * HALF[dtype] * one.float().abs() + 2.0 ** -14 * float(one.float().abs().max())    # (both within their E of one value)
            assert ((many.view(3, T, -1)[:, t].float() - one.float()).abs() <= tol).all()
        same = lambda x, y: torch.equal(x.view(torch.uint8), y.view(torch.uint8))
        assert same(a.k, b.k) and same(a.v, b.v)


# ------------------------------------------------------------------------------------------------ eviction
def _evict_reference(w, n, budget, recent):
    """Slots kept by one row and head, by the definition: w float list of n weights."""
    if n <= budget:
        return list(range(n)) + [-1] * (budget - n)
    A, old = budget - recent, n - recent
    key = lambda s: (0 if w[s] != w[s] else 1, 0.0 if w[s] != w[s] else -w[s], s)        # NaN above everything, then the greatest, then the lowest
    best = set(sorted(range(old), key=key)[:A])
    late = [s for s in sorted(best) if s >= A]
    out = [s if s in best else late.pop(0) for s in range(A)]
    return out + list(range(n - recent, n))


EVICT = [
    # dtype, Hkv, d, page, lens, budget, recent
    (torch.bfloat16, 2, 128, 16, [100, 64, 65, 0, -1, 200], 64, 16),
    (torch.float32, 3, 100, 8, [100, 33, 32, 500], 32, 0),
    (torch.bfloat16, 2, 64, 4, [100, 41, 40, 39], 40, 40),
    (torch.bfloat16, 1, 36, 16, [300, 17], 1, 1),
    (torch.float32, 1, 4, 16, [300, 17, 2], 1, 0),
    (torch.bfloat16, 4, 192, 64, [1500, 1024, 700], 600, 100),
    (torch.bfloat16, 1, 512, 32, [3500, 2049], 2048, 7),
    (torch.bfloat16, 2, 64, 16, [50, 60], 100, 10),
    (torch.float32, 2, 64, 128, [20000, 16384, 9000], 8000, 900),
    (torch.bfloat16, 1, 8, 1024, [70000, 66000, 5], 30000, 1000),              # more slots than a workgroup's registers hold
    (torch.bfloat16, 1, 12, 256, [40000, 33000], 32000, 31000),                # a long shift that overlaps itself
    (torch.bfloat16, 2, 128, 16, [4000, 2100], 2000, 0),
    (torch.float32, 1, 128, 64, [3001, 3002], 3000, 2999),
]


@pytest.mark.parametrize("kind", ["spread", "ties", "odd"])
@pytest.mark.parametrize("case", EVICT, ids=lambda c: f"{str(c[0])[6:]}-Hkv{c[1]}-d{c[2]}-page{c[3]}-budget{c[5]}-recent{c[6]}")
def test_evict_against_the_definition(case, kind):
    from multimodal_amd import ops
    dtype, Hkv, d, page, lens, budget, recent = case
    g = torch.Generator().manual_seed(41)
    B = len(lens)
    c = Cache(41, dtype, B, Hkv, d, page, lens, weights=True)
    ws = []
    for b, n in enumerate(lens):
        n = max(n, 0)
        w = torch.rand(Hkv, n, generator=g).exp()
        if kind == "ties":
            w = torch.randint(0, 3, (Hkv, n), generator=g).float()
        if kind == "odd" and n:
            pick = torch.randint(0, 12, (Hkv, n), generator=g)
            for i, x in enumerate((float("nan"), float("inf"), -float("inf"), 0.0, -0.0, -1.5, 1e-45, -float("nan"))):
                w[pick == i] = x
        ws.append(w)
        if n:
            c.put(c.k, b, n, _randn(g, Hkv, n, d)); c.put(c.v, b, n, _randn(g, Hkv, n, d)); c.put(c.w, b, n, w)
    before = (c.k.clone(), c.v.clone(), c.w.clone())
    n_dev = torch.tensor(lens, dtype=torch.int32, device=DEV)
    kept = ops.paged_evict(c.k, c.v, c.w, c.table, n_dev, budget, recent)
    assert kept.dtype == torch.int32 and kept.shape == (B, Hkv, budget)
    assert n_dev.tolist() == [min(x, budget) for x in lens]
    touched = torch.zeros(c.n_pages, Hkv, page, dtype=torch.bool)
    for b, n in enumerate(lens):
        for h in range(Hkv):
            want = _evict_reference(ws[b][h].tolist(), max(n, 0), budget, recent)
            assert kept[b, h].tolist() == want, (b, h)
            if n > budget:
                src = torch.tensor(want)
                pg, off = c.table[b].cpu().long()[src // page], src % page
                to = torch.arange(budget)
                pt, ot = c.table[b].cpu().long()[to // page], to % page
                for got, old in ((c.k, before[0]), (c.v, before[1]), (c.w, before[2])):
                    x, y = got[pt.to(DEV), h, ot.to(DEV)], old[pg.to(DEV), h, off.to(DEV)]
                    assert torch.equal(x.contiguous().view(torch.uint8), y.contiguous().view(torch.uint8)), (b, h)
                touched[pt, h, ot] = True
    keep = (~touched).to(DEV)
    for got, old in ((c.k, before[0]), (c.v, before[1]), (c.w, before[2])):
        assert torch.equal(got[keep].view(torch.uint8), old[keep].view(torch.uint8)), "slots behind the budget or of other rows were touched"


def test_evict_pages_the_table_does_not_hold():
    """Slots on pages outside the pool count as the lowest and are never touched; rows longer than their table count as their table's slots."""
    from multimodal_amd import ops
    c = Cache(43, torch.bfloat16, 2, 1, 64, 16, [160, 160], weights=True, garbage=0.0)
    g = torch.Generator().manual_seed(43)
    ws = []
    for b in range(2):
        w = torch.rand(1, 160, generator=g) + 0.5
        c.put(c.k, b, 160, _randn(g, 1, 160, 64)); c.put(c.v, b, 160, _randn(g, 1, 160, 64)); c.put(c.w, b, 160, w)
        ws.append(w[0])
    c.table[0, 4] = -1                                    # slots 64 .. 79, behind the kept region
    ws[0][64:80] = -math.inf
    n = torch.tensor([160, 1000], dtype=torch.int32, device=DEV)
    kept = ops.paged_evict(c.k, c.v, c.w, c.table, n, 60, 12)
    assert n.tolist() == [60, 60]
    assert kept[0, 0].tolist() == _evict_reference(ws[0].tolist(), 160, 60, 12)
    assert kept[1, 0].tolist() == _evict_reference(ws[1].tolist(), 160, 60, 12)


def test_evict_many_slots_and_missing_pages():
    """Moves and shift side by side, with pages missing among the holes, the survivors, the slots the shift overwrites and those it takes: what has
    a source and a target moves, everything else stays."""
    from multimodal_amd import ops
    n_slots, budget, recent, page, d = [4000, 2300], 2000, 600, 16, 128
    g = torch.Generator().manual_seed(44)
    c = Cache(44, torch.bfloat16, 2, 2, d, page, n_slots, weights=True, garbage=0.0)
    ws = []
    for b, n in enumerate(n_slots):
        w = torch.rand(2, n, generator=g) + 0.5
        c.put(c.k, b, n, _randn(g, 2, n, d)); c.put(c.v, b, n, _randn(g, 2, n, d)); c.put(c.w, b, n, w)
        ws.append(w)
    for b, entry in ((0, 4), (0, 88), (0, 110), (0, 150), (0, 225), (1, 3), (1, 90), (1, 107), (1, 130)):
        c.table[b, entry] = -1 if entry % 2 else c.n_pages
        s = slice(entry * page, (entry + 1) * page)
        ws[b][:, s] = -math.inf
    before = (c.k.clone(), c.v.clone(), c.w.clone())
    n_dev = torch.tensor(n_slots, dtype=torch.int32, device=DEV)
    kept = ops.paged_evict(c.k, c.v, c.w, c.table, n_dev, budget, recent)
    assert n_dev.tolist() == [budget, budget]
    want = [x.clone() for x in before]
    table = c.table.cpu().long()
    for b, n in enumerate(n_slots):
        for h in range(2):
            ref = _evict_reference(ws[b][h].tolist(), n, budget, recent)
            assert kept[b, h].tolist() == ref, (b, h)
            src, to = torch.tensor(ref), torch.arange(budget)
            ps, pt = table[b][src // page], table[b][to // page]
            both = (ps >= 0) & (ps < c.n_pages) & (pt >= 0) & (pt < c.n_pages)
            ps, pt, os, ot = ps[both].to(DEV), pt[both].to(DEV), (src % page)[both].to(DEV), (to % page)[both].to(DEV)
            for x, y in zip(want, before):
                x[pt, h, ot] = y[ps, h, os]
    for x, y in zip((c.k, c.v, c.w), want):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


def _evict_large(seed, dtype, B, Hkv, d, page, lens, budget, recent, missing=0.0):
    """An eviction of many slots: kept by a stable sort, the pools bit by bit, everything on the GPU.  Weights are distinct but for a tenth;
    missing: this share of the table's entries names no page."""
    from multimodal_amd import ops
    g = torch.Generator(device=DEV).manual_seed(seed)
    width = -(-max(lens) // page)
    n_pages = B * width + 3
    table = torch.randperm(n_pages, generator=g, device=DEV)[: B * width].view(B, width)
    there = torch.rand(B, width, generator=g, device=DEV) >= missing
    k = torch.empty(n_pages, Hkv, page, d, dtype=dtype, device=DEV).normal_(generator=g)
    v = torch.empty_like(k).normal_(generator=g)
    w = torch.rand(n_pages, Hkv, page, generator=g, device=DEV)
    w[w < 0.1] = 0.5
    before = (k.clone(), v.clone(), w.clone())
    n = torch.tensor(lens, dtype=torch.int32, device=DEV)
    kept = ops.paged_evict(k, v, w, torch.where(there, table, -1).int(), n, budget, recent)
    assert n.tolist() == [min(x, budget) for x in lens]
    A, j = budget - recent, torch.arange(budget, device=DEV)
    for b, m in enumerate(lens):
        if m <= budget:
            assert (kept[b] == torch.where(j < m, j, -1)).all(), b
            continue
        on = there[b].repeat_interleave(page)
        ws = before[2][table[b]].transpose(0, 1).reshape(Hkv, -1).masked_fill(~on, -math.inf)[:, : m - recent]
        best = torch.zeros_like(ws, dtype=torch.bool).scatter_(1, ws.sort(dim=1, descending=True, stable=True).indices[:, :A], True)
        want = torch.cat((j[:A].expand(Hkv, A), torch.arange(m - recent, m, device=DEV).expand(Hkv, recent)), 1).clone()
        want[:, :A][~best[:, :A]] = best[:, A:].nonzero()[:, 1] + A                      # row by row, holes and survivors alike in order
        assert torch.equal(kept[b].long(), want), b
        h, to = (on[want] & on[j]).nonzero(as_tuple=True)
        src = want[h, to]
        for y in before:
            y[table[b][to // page], h, to % page] = y[table[b][src // page], h, src % page].clone()
    for x, y in zip((k, v, w), before):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 128), (torch.float32, 100), (torch.bfloat16, 100)])
def test_evict_past_the_last_level_cache(dtype, d):
    """Pools of more than 256 MB: what moves goes past the cache (16- and 8-byte pieces)."""
    lens = [4096, 4000, 2049, 2048, 1, 0] + [3000 + 37 * i for i in range(26)]
    assert 32 * 8 * 4096 * d * 2 * dtype.itemsize > 256 << 20
    _evict_large(45, dtype, 32, 8, d, 64, lens, 2048, 100)


@pytest.mark.parametrize("dtype,Hkv,d,page,longest,budget,recent", [
    (torch.bfloat16, 8, 64, 16, 300, 64, 16), (torch.float32, 2, 100, 16, 200, 40, 0), (torch.bfloat16, 8, 128, 8, 90, 33, 33),
    (torch.bfloat16, 4, 36, 16, 2000, 100, 20), (torch.bfloat16, 1, 8, 1024, 12000, 60, 5), (torch.bfloat16, 1, 4, 1024, 40000, 300, 30),
    (torch.bfloat16, 1, 4, 1024, 70000, 300, 30)])
def test_evict_many_rows(dtype, Hkv, d, page, longest, budget, recent):
    """Rows and heads that fill the card, of every length: a workgroup each does it all."""
    B = 800 // min(Hkv, 4) + 7
    lens = [1 + (longest - 1) * i // (B - 1) for i in range(B)]
    _evict_large(46, dtype, B, Hkv, d, page, lens[::-1], budget, recent)
    _evict_large(47, dtype, B, Hkv, d, page, lens, budget, recent, missing=0.1)


# ------------------------------------------------------------------------------------------------ together
def _simulate(dtype, lens, steps, budget, recent, stable, seed=50):
    """Prompts, steps with weights, an eviction whenever a row passes its budget: the operators against a 64-bit simulation that keeps each row's
    slots as lists.  Every step is checked against the definition on what is stored; evictions against the simulated weights' order."""
    from multimodal_amd import ops
    Hkv, G, d, rot, page = 2, 2, 64, 32, 8
    H, B = Hkv * G, len(lens)
    g = torch.Generator().manual_seed(seed)
    room = max(max(lens), budget) + steps + 1
    c = Cache(seed, dtype, B, Hkv, d, page, [room] * B, weights=True)
    tabs = _tables(rot, 256)
    S = max(lens)
    kv = _randn(g, B, S, 2 * Hkv * d, dtype=dtype).to(DEV)
    n = torch.tensor(lens, dtype=torch.int32, device=DEV)
    ops.paged_cache_fill(kv[..., : Hkv * d], kv[..., Hkv * d:], c.k, c.v, c.table, rot, *tabs, counts=n, weights=c.w)
    pos = n.clone()
    evictions = 0
    for t in range(steps):
        x = _randn(g, B, (H + 2 * Hkv) * d, dtype=dtype).to(DEV)
        q, k, v = x[:, : H * d], x[:, H * d: (H + Hkv) * d], x[:, (H + Hkv) * d:]
        before = (c.k.clone(), c.v.clone(), c.w.clone())
        o = ops.paged_decode_attn(q, k, v, c.k, c.v, c.table, n, H, rot, *tabs, stable, positions=pos, weights=c.w)
        _check_step(c, before, q, k, v, n.tolist(), H, rot, tabs, stable, pos.tolist(), o)
        n.add_(1); pos.add_(1)
        if t % 3 == 2:
            old = n.tolist()
            ws = [c.rows(c.w, b, m) for b, m in enumerate(old)]
            ks = [c.rows(c.k, b, m) for b, m in enumerate(old)]
            kept = ops.paged_evict(c.k, c.v, c.w, c.table, n, budget, recent)
            for b, m in enumerate(old):
                for h in range(Hkv):
                    want = _evict_reference(ws[b][h].tolist(), m, budget, recent)
                    assert kept[b, h].tolist() == want
                    live = [s for s in want if s >= 0]
                    assert torch.equal(c.rows(c.k, b, len(live))[h], ks[b][h][live])
            evictions += sum(m > budget for m in old)
    return evictions


@pytest.mark.parametrize("stable", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_fill_attend_evict_together(dtype, stable):
    assert _simulate(dtype, [5, 20, 33, 1], steps=14, budget=24, recent=6, stable=stable) >= 6


def test_captured_steps_replayed_on_two_streams():
    """Two graphs captured on one stream, each a step and an eviction of its own rows, replayed beside each other several times with eager work
    between: every replay equals the eager result."""
    from multimodal_amd import ops
    lens = [700, 30, 2049]
    made = [_filled(60 + i, torch.bfloat16, 3, 2, 2, 64, 16, lens, weights=True) for i in range(2)]
    base = [(c.k.clone(), c.v.clone(), c.w.clone()) for c, *_ in made]
    n0 = torch.tensor(lens, dtype=torch.int32, device=DEV)

    def step(c, q, k, v, n):
        o = ops.paged_decode_attn(q, k, v, c.k, c.v, c.table, n, 4, 0, None, None, False, weights=c.w)
        n.add_(1)
        kept = ops.paged_evict(c.k, c.v, c.w, c.table, n, 640, 32)
        return o, kept

    def reset(i, n):
        c = made[i][0]
        c.k.copy_(base[i][0]); c.v.copy_(base[i][1]); c.w.copy_(base[i][2]); n.copy_(n0)
    ns = [n0.clone(), n0.clone()]
    want = []
    for i in range(2):
        o, kept = step(*made[i], ns[i])
        want.append((o.clone(), kept.clone(), made[i][0].k.clone(), made[i][0].w.clone()))
        reset(i, ns[i])
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    graphs, outs = [], []
    with torch.cuda.stream(s):
        for i in range(2):
            g = torch.cuda.CUDAGraph()
            g.capture_begin()
            outs.append(step(*made[i], ns[i]))
            g.capture_end()
            graphs.append(g)
    torch.cuda.synchronize()
    others = [torch.cuda.Stream(), torch.cuda.Stream()]
    junk = torch.randn(512, 512, device=DEV)
    for _ in range(4):
        for i in range(2):
            reset(i, ns[i])
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(others[i]):
                graphs[i].replay()
        junk = junk @ junk.t() / 512
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(outs[i][0], want[i][0]) and torch.equal(outs[i][1], want[i][1])
            same = lambda a, b: torch.equal(a.view(torch.uint8), b.view(torch.uint8))
            assert same(made[i][0].k, want[i][2]) and same(made[i][0].w, want[i][3])


def test_two_calls_at_once_on_two_streams():
    from multimodal_amd import ops
    sets = [_filled(70 + i, torch.bfloat16, 4, 2, 4, 128, 32, [3000, 1, 900, 4000]) for i in range(2)]
    n = torch.tensor([3000, 1, 900, 4000], dtype=torch.int32, device=DEV)
    want = [ops.paged_decode_attn(q, k, v, c.k, c.v, c.table, n, 8, 0, None, None, False) for c, q, k, v in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        got = []
        for s, (c, q, k, v) in zip(streams, sets):
            with torch.cuda.stream(s):
                got.append(ops.paged_decode_attn(q, k, v, c.k, c.v, c.table, n, 8, 0, None, None, False))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


# ------------------------------------------------------------------------------------------------ refusals
def test_refusals():
    from multimodal_amd import ops
    c, q, k, v = _filled(80, torch.bfloat16, 2, 2, 2, 64, 16, [5, 6], weights=True)
    n = torch.tensor([5, 6], dtype=torch.int32, device=DEV)
    tabs = _tables(32, 64)
    ok = dict(q=q, k_new=k, v_new=v, kpool=c.k, vpool=c.v, page_table=c.table, lengths=n, H=4, rot=32, cos_t=tabs[0], sin_t=tabs[1], stablemax=False)
    before = c.k.clone()
    bad = [
        (dict(q=q.float()), RuntimeError), (dict(q=q[:, :-1]), RuntimeError), (dict(q=q.cpu()), RuntimeError), (dict(k_new=None), RuntimeError),
        (dict(k_new=k[:1]), RuntimeError), (dict(H=3), RuntimeError), (dict(H=0), RuntimeError), (dict(rot=33), RuntimeError),
        (dict(rot=66), RuntimeError), (dict(rot=-2), RuntimeError), (dict(cos_t=None), RuntimeError), (dict(cos_t=tabs[0][:, :8]), RuntimeError),
        (dict(lengths=n.long()), TypeError), (dict(lengths=n[:1]), RuntimeError), (dict(lengths=n.cpu()), RuntimeError),
        (dict(page_table=c.table.long()), RuntimeError), (dict(page_table=c.table[0]), RuntimeError), (dict(page_table=c.table.t()), RuntimeError),
        (dict(vpool=c.k), RuntimeError), (dict(vpool=c.v.float()), TypeError), (dict(kpool=c.k[:, :, :12]), RuntimeError),
        (dict(kpool=c.k[:, :, :12].contiguous(), vpool=c.v[:, :, :12].contiguous()), RuntimeError),
        (dict(kpool=c.k.half(), vpool=c.v.half()), TypeError), (dict(weights=c.w.double()), TypeError), (dict(weights=c.w[:1]), RuntimeError),
        (dict(positions=n.long()), TypeError), (dict(q=q[:, ::2]), RuntimeError),
    ]
    for change, kind in bad:
        with pytest.raises(kind):
            ops.paged_decode_attn(**{**ok, **change})
    wide = torch.zeros(2, 2, 16, 516, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(RuntimeError, match="head_dim"):
        ops.paged_cache_fill(torch.zeros(2, 1, 1032, dtype=torch.bfloat16, device=DEV), torch.zeros(2, 1, 1032, dtype=torch.bfloat16, device=DEV),
                             wide, wide.clone(), c.table, 0, None, None)
    with pytest.raises(RuntimeError, match="aligned"):
        flat = torch.zeros(c.k.numel() + 4, dtype=torch.bfloat16, device=DEV)
        ops.paged_decode_attn(**{**ok, "kpool": flat[4:].view_as(c.k)})
    with pytest.raises(RuntimeError, match="backward"):
        ops.paged_decode_attn(**{**ok, "q": q.clone().requires_grad_()})
    for budget, recent in ((0, 0), (4, 5), (4, -1)):
        with pytest.raises(RuntimeError, match="budget"):
            ops.paged_evict(c.k, c.v, c.w, c.table, n, budget, recent)
    with pytest.raises(RuntimeError):
        ops.paged_evict(c.k, c.v, None, c.table, n, 4, 1)
    kv = torch.zeros(2, 3, 128, dtype=torch.bfloat16, device=DEV)
    for change in (dict(v=kv[:, :2]), dict(k=kv[0]), dict(k=kv.float()), dict(start=n.long()), dict(counts=n[:1]), dict(rot=3)):
        with pytest.raises((RuntimeError, TypeError)):
            ops.paged_cache_fill(**{**dict(k=kv, v=kv, kpool=c.k, vpool=c.v, page_table=c.table, rot=0, cos_t=None, sin_t=None), **change})
    torch.cuda.synchronize()
    assert torch.equal(before.view(torch.uint8), c.k.view(torch.uint8))


def test_nothing_to_do():
    """No rows, no tokens."""
    from multimodal_amd import ops
    c, q, k, v = _filled(81, torch.bfloat16, 2, 2, 2, 64, 16, [5, 6], weights=True)
    n = torch.tensor([5, 6], dtype=torch.int32, device=DEV)
    assert ops.paged_decode_attn(q[:0], k[:0], v[:0], c.k, c.v, c.table[:0], n[:0], 4, 0, None, None, False).shape == (0, 256)
    ops.paged_cache_fill(torch.zeros(2, 0, 128, dtype=torch.bfloat16, device=DEV), torch.zeros(2, 0, 128, dtype=torch.bfloat16, device=DEV), c.k, c.v,
                         c.table, 0, None, None)
    assert ops.paged_evict(c.k, c.v, c.w, c.table[:0], n[:0], 4, 1).shape == (0, 2, 4)
