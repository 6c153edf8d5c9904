"""GPU parity of attention behind a shared prefix against the formula in float64.

Tolerances, elementwise, with u = half a step of the type (2^-8 bf16, 2^-11 fp16), A = sum p |v| / sum p (at
least |o|) and X = max_j scale sum_d |q_d k_jd|:
  * a score is a sum of D products, of which each step rounds or truncates by at most 2^-22 of the magnitudes
    added: D 2^-22 X; its scaling into the log2 domain, the subtraction of a maximum of at most X and the
    exponential add 2^-20 (1 + X) relative: E = D 2^-22 X + 2^-20 (1 + X) bounds p's relative error;
  * rounding p for the product: u A; rounding the result: u A; E in numerator and denominator: 2 E A. fp16 cannot
    hold p below 2^-31 of the maximum: 2^-31 max |v| for each of N keys;
  * merging n parts scales and adds n terms: 2 n 2^-22 A. lse: E + 2^-20 (1 + |lse|).
"""
from __future__ import annotations

import math

import pytest

from conftest import cuda_available

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not cuda_available(), reason="needs a CUDA device")]

HALF_STEP = {"bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}
PARTS = 512  # more parts than any call here has


def make(batch, heads, kv_heads, tokens, dim, prefix, cache, dtype="bfloat16", seed=0, std=1.0):
    import torch

    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = getattr(torch, dtype)

    def one(*shape):
        return (torch.randn(*shape, device="cuda", generator=gen) * std).to(dt)

    return (one(batch, heads, tokens, dim), one(kv_heads, prefix, dim), one(kv_heads, prefix, dim),
            one(batch, kv_heads, cache, dim), one(batch, kv_heads, cache, dim))


def reference(q, pk, pv, k, v, lens, scale):
    """(o, lse, tolerance of o, tolerance of lse) in float64, query by query."""
    import torch

    b, h, t, d = q.shape
    hk, cache = k.shape[1], k.shape[2]
    per = h // hk
    u = HALF_STEP[str(q.dtype)[6:]]
    o = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.full(q.shape[:3], -math.inf, dtype=torch.float64, device=q.device)
    tol, tol_lse = torch.zeros_like(o), torch.zeros_like(lse)
    for i in range(b):
        n = cache if lens is None else max(0, min(int(lens[i]), cache))
        for j in range(t):
            own = n - t + j + 1
            if own < 1:
                continue
            kk = torch.cat([pk, k[i, :, :own]], 1).double()
            vv = torch.cat([pv, v[i, :, :own]], 1).double()
            qq = q[i, :, j].double().view(hk, per, d)
            s = torch.einsum("gpd,gkd->gpk", qq, kk) * scale
            top = s.amax(-1, keepdim=True)
            p = torch.exp(s - torch.where(torch.isinf(top), 0.0, top))
            total = p.sum(-1, keepdim=True)
            p = p / torch.where(total == 0, 1.0, total)
            x = (torch.einsum("gpd,gkd->gpk", qq.abs(), kk.abs()) * scale).nan_to_num(posinf=0.0).amax(-1, keepdim=True)
            e = d * 2.0 ** -22 * x + 2.0 ** -20 * (1 + x)
            mean = torch.matmul(p, vv.abs())
            o[i, :, j] = torch.matmul(p, vv).view(h, d)
            lse[i, :, j] = (top + total.log()).view(h)
            tol[i, :, j] = ((2 * u + 2 * e + PARTS * 2.0 ** -21) * mean
                            + kk.shape[1] * 2.0 ** -31 * vv.abs().amax()).view(h, d)
            tol_lse[i, :, j] = (e + 2.0 ** -20 * (1 + lse[i, :, j].view(hk, per, 1).abs().nan_to_num(posinf=0.0))).view(h)
    return o, lse, tol, tol_lse


def check(args, lens=None, scale=None, got=None):
    import torch

    import neptune_opt_b200 as NB

    scale = 1.0 / math.sqrt(args[0].shape[-1]) if scale is None else scale
    o, lse = NB.prefix_attention(*args, lens, scale=scale, return_lse=True) if got is None else got
    ro, rl, tol, tol_lse = reference(*args, lens, scale)
    assert o.dtype == args[0].dtype and o.shape == args[0].shape and o.is_contiguous()
    off = (o.double() - ro).abs()
    assert bool((off <= tol).all()), f"o off by up to {(off - tol).amax():.3e} beyond its bound"
    dead = torch.isinf(rl)
    assert torch.equal(torch.isinf(lse), dead) and bool((lse[dead] < 0).all())
    off = (lse.double() - rl).abs()[~dead]
    assert bool((off <= tol_lse[~dead]).all()), f"lse off by up to {(off - tol_lse[~dead]).amax():.3e} beyond its bound"
    return o, lse


def lens_of(*values):
    import torch

    return torch.tensor(values, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv_heads,tokens", [(1, 1, 1), (8, 2, 1), (6, 2, 3), (5, 1, 7), (16, 1, 4)])
def test_against_the_formula(dtype, dim, heads, kv_heads, tokens):
    check(make(3, heads, kv_heads, tokens, dim, 333, 150, dtype), lens_of(150, 77, tokens))


@pytest.mark.parametrize("prefix", [0, 1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 1000])
@pytest.mark.parametrize("cache", [1, 16, 65])
def test_key_counts_around_the_tiles(prefix, cache):
    check(make(2, 8, 2, 1, 128, prefix, cache, seed=prefix + cache))


def test_lengths_from_nothing_to_full():
    """Free slots, a sequence shorter than the new tokens, and lengths outside the cache (read as clamped)."""
    import torch

    args = make(9, 8, 4, 3, 128, 100, 64)
    lens = lens_of(0, 1, 2, 3, 4, 63, 64, 99, -5)
    o, lse = check(args, lens)
    assert not o[0].any() and not o[8].any() and bool(torch.isinf(lse[0]).all())
    assert not o[1][:, :2].any() and o[1][:, 2].any()


@pytest.mark.parametrize("prefix", [0, 200])
def test_a_cache_without_room(prefix):
    """No own tokens at all: every query is one of a free slot."""
    import torch

    import neptune_opt_b200 as NB

    o, lse = NB.prefix_attention(*make(2, 4, 2, 1, 64, prefix, 0), return_lse=True)
    assert not o.any() and bool(torch.isinf(lse).all())


def test_what_a_cache_holds_behind_a_sequence_does_not_matter():
    import torch

    import neptune_opt_b200 as NB

    q, pk, pv, k, v = make(4, 8, 2, 2, 128, 130, 90)
    lens = lens_of(90, 33, 0, 2)
    want = check((q, pk, pv, k, v), lens)
    for junk in (math.nan, math.inf, -math.inf):
        k2, v2 = k.clone(), v.clone()
        for i, n in enumerate(lens.tolist()):
            k2[i, :, n:] = junk
            v2[i, :, n:] = junk
        got = NB.prefix_attention(q, pk, pv, k2, v2, lens, return_lse=True)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_keys_that_no_query_can_weigh():
    """Scores of -inf have no weight, in the prefix and in a cache; a row of them alone is an empty row."""
    import torch

    import neptune_opt_b200 as NB

    q, pk, pv, k, v = make(2, 4, 2, 1, 64, 140, 50)
    q[..., 0] = q[..., 0].abs() + 0.5
    pk[:, 3:130, 0] = -math.inf
    k[1, :, ::2, 0] = -math.inf
    o, lse = NB.prefix_attention(q, pk, pv, k, v, return_lse=True)
    clean = reference(q[:1], torch.cat([pk[:, :3], pk[:, 130:]], 1), torch.cat([pv[:, :3], pv[:, 130:]], 1), k[:1], v[:1], None, 0.125)
    assert bool(((o[:1].double() - clean[0]).abs() <= clean[2]).all())
    assert bool(((lse[:1].double() - clean[1]).abs() <= clean[3]).all())
    pk[..., 0] = k[..., 0] = -math.inf
    o, lse = NB.prefix_attention(q, pk, pv, k, v, return_lse=True)
    assert not o.any() and bool((lse == -math.inf).all())


def test_a_nan_key_reaches_the_rows_that_see_it():
    import torch

    import neptune_opt_b200 as NB

    q, pk, pv, k, v = make(3, 4, 2, 1, 128, 300, 70)
    k[1, 0, 5] = math.nan
    o, lse = NB.prefix_attention(q, pk, pv, k, v, return_lse=True)
    bad = torch.zeros(3, 4, dtype=torch.bool, device="cuda")
    bad[1, :2] = True
    assert torch.equal(torch.isnan(o).all(-1)[..., 0], bad) and torch.equal(torch.isnan(lse)[..., 0], bad)
    pk[1, 200] = math.nan
    bad[:, 2:] = True
    o, lse = NB.prefix_attention(q, pk, pv, k, v, return_lse=True)
    assert torch.equal(torch.isnan(o).all(-1)[..., 0], bad) and torch.equal(torch.isnan(lse)[..., 0], bad)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_scores_far_apart(dtype):
    """Maxima that grow along the keys (the running maximum moves many times) and scores of several hundred."""
    import torch

    q, pk, pv, k, v = make(2, 8, 2, 1, 128, 1500, 200, dtype)
    ramp = torch.linspace(0.1, 6.0, 1500, device="cuda")[None, :, None].to(q.dtype)
    check((q, pk * ramp, pv, k * 8, v))
    check((q, pk * ramp.flip(1), pv, k * 0.01, v))


def test_many_unlikely_keys_in_fp16():
    """One key far above 60000 others that together weigh as much: none of them may vanish in fp16."""
    import torch

    q, pk, pv, k, v = make(1, 2, 1, 1, 64, 60000, 1, "float16")
    q.fill_(1.0)
    pk.zero_()
    pv.fill_(1.0)
    k.fill_(11.0 / 8.0)  # score 64 * 11/8 / 8 = 11, e^11 = 59874 against 60000 keys of weight 1
    v.fill_(-1.0)
    o, _ = check((q, pk, pv, k, v))
    assert bool((o.abs() < 0.01).all())


@pytest.mark.parametrize("batch,heads,kv_heads,tokens,prefix,cache", [
    (64, 32, 8, 1, 700, 100), (40, 16, 2, 3, 500, 40), (17, 8, 8, 1, 3001, 33), (1, 64, 1, 1, 2000, 2000),
    (130, 4, 4, 1, 257, 9), (33, 8, 1, 1, 1025, 5), (3, 40, 8, 8, 999, 130)])
def test_many_query_rows(batch, heads, kv_heads, tokens, prefix, cache):
    """More query rows per key/value head than one tile holds, whole and ragged tiles."""
    lens = [max(0, cache - 3 * i) for i in range(batch)]
    check(make(batch, heads, kv_heads, tokens, 128, prefix, cache, seed=batch), lens_of(*lens))


@pytest.mark.parametrize("dim", [64, 128])
def test_layouts(dim):
    """Tensors as models hold them: sequence before heads, slices of one projection, a longer cache's front, an
    unaligned base, and an expanded batch (the last two are copied first)."""
    import torch

    import neptune_opt_b200 as NB

    b, h, hk, p, s = 3, 4, 2, 100, 40
    q, pk, pv, k, v = make(b, h, hk, 1, dim, p, s)
    lens = lens_of(40, 7, 21)
    want = check((q, pk, pv, k, v), lens)

    def same(*args):
        got = NB.prefix_attention(*args, lens, return_lse=True)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])

    swap = lambda t: t.transpose(-3, -2).contiguous().transpose(-3, -2)  # noqa: E731
    same(swap(q), swap(pk), swap(pv), swap(k), swap(v))
    qkv = torch.cat([q, q, k[:, :, :1], v[:, :, :1]], 1)
    same(qkv[:, :h], pk, pv, k, v)
    long = torch.full((b, hk, 3 * s, dim), math.nan, device="cuda", dtype=q.dtype)
    long[:, :, :s] = k
    same(q, pk, pv, long[:, :, :s], v)
    kv = torch.stack([pk, pv], 2)
    same(q, kv[:, :, 0], kv[:, :, 1], k, v)
    shift = torch.empty(k.numel() + 1, device="cuda", dtype=k.dtype)[1:].view(k.shape)
    shift.copy_(k)
    same(q, pk, pv, shift, v)
    one = k[:1].expand(b, -1, -1, -1)
    got = NB.prefix_attention(q, pk, pv, one, one, lens, return_lse=True)
    ref = NB.prefix_attention(q, pk, pv, one.contiguous(), one.contiguous(), lens, return_lse=True)
    assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])


def test_offsets_past_32_bits():
    """A cache of which the later sequences lie more than 2^32 bytes, and 2^31 elements, from its start."""
    import torch

    q, pk, pv, k, v = make(3, 2, 1, 1, 128, 20, 30)
    room = torch.zeros(3, 1, 9_000_000, 128, device="cuda", dtype=q.dtype)  # 6.9 GB; its batch stride is 1.15e9 elements
    room[:, :, -30:] = k
    check((q, pk, pv, room[:, :, -30:], v))


# Calls of few keys and sequences run as one kernel; what follows does not: more than 16 query rows a key/value
# head of a sequence, or more keys than few units take on.
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("batch,heads,kv_heads,tokens,prefix,cache", [
    (1, 1, 1, 1, 333, 2100), (2, 8, 2, 2, 2000, 333), (3, 16, 1, 1, 100, 2500), (3, 24, 1, 1, 333, 150), (2, 6, 2, 7, 40, 90),
    (2, 4, 2, 1, 0, 3001), (2, 4, 2, 1, 3001, 3), (2, 33, 1, 1, 17, 1), (9, 24, 1, 2, 0, 64)])
def test_parts_in_memory(dtype, dim, batch, heads, kv_heads, tokens, prefix, cache):
    args = make(batch, heads, kv_heads, tokens, dim, prefix, cache, dtype, seed=prefix)
    check(args)
    check(args, lens_of(*[(cache, 0, tokens, cache // 2, 1, 99999, -3, 16, 17)[i] for i in range(batch)]))


def test_empty_rows_and_junk_with_parts_in_memory():
    import torch

    import neptune_opt_b200 as NB

    q, pk, pv, k, v = make(5, 48, 2, 1, 128, 140, 90)
    lens = lens_of(90, 33, 0, 1, 17)
    want = check((q, pk, pv, k, v), lens)
    assert not want[0][2].any()
    for junk in (math.nan, math.inf, -math.inf):
        k2, v2 = k.clone(), v.clone()
        for i, n in enumerate(lens.tolist()):
            k2[i, :, n:] = junk
            v2[i, :, n:] = junk
        got = NB.prefix_attention(q, pk, pv, k2, v2, lens, return_lse=True)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    q[..., 0] = q[..., 0].abs() + 0.5
    pk[..., 0] = -math.inf
    k[..., 0] = -math.inf
    o, lse = NB.prefix_attention(q, pk, pv, k, v, return_lse=True)
    assert not o.any() and bool((lse == -math.inf).all())
    k[1, 0, 5] = math.nan
    o, lse = NB.prefix_attention(q, pk, pv, k, v, return_lse=True)
    assert bool(torch.isnan(o[1, :24]).all()) and not o[1, 24:].any() and not o[0].any()


@pytest.mark.parametrize("dim", [64, 128])
def test_one_kernel_and_parts_in_memory_agree(dim):
    """The first sequences alone and the whole batch, which has more units than SMs: both within the bounds, in layouts
    of rows that lie apart."""
    import torch

    import neptune_opt_b200 as NB

    q, pk, pv, k, v = make(200, 8, 4, 1, dim, 301, 1500)
    q, k, v = q.transpose(0, 1).contiguous().transpose(0, 1), k.transpose(1, 2).contiguous().transpose(1, 2), v
    lens = torch.randint(0, 1501, (200,), dtype=torch.int32, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    for n in (1, 7, 40, 200):
        o, lse = NB.prefix_attention(q[:n], pk, pv, k[:n], v[:n], lens[:n], return_lse=True)
        some = slice(max(0, n - 3), n)
        check((q[some], pk, pv, k[some], v[some]), lens[some], got=(o[some], lse[some]))


def test_other_scales():
    check(make(2, 4, 2, 1, 128, 90, 20), scale=1.0)
    check(make(2, 4, 2, 1, 128, 90, 20, std=3.0), scale=1e-4)


def test_runs_are_alike():
    import torch

    import neptune_opt_b200 as NB

    args, lens = make(5, 32, 8, 1, 128, 5000, 700), lens_of(700, 3, 0, 650, 128)
    first = NB.prefix_attention(*args, lens, return_lse=True)
    for _ in range(5):
        again = NB.prefix_attention(*args, lens, return_lse=True)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
    assert torch.equal(NB.prefix_attention(*args, lens), first[0])


def test_as_one_cache():
    """The prefix in front of each sequence's own cache gives the same attention."""
    import torch

    import neptune_opt_b200 as NB

    q, pk, pv, k, v = make(4, 8, 2, 2, 128, 300, 100)
    lens = lens_of(100, 50, 2, 99)
    o, lse = check((q, pk, pv, k, v), lens)
    whole_k, whole_v = (torch.cat([p[None].expand(4, -1, -1, -1), c], 2) for p, c in ((pk, k), (pv, v)))
    empty = pk[:, :0]
    o2, lse2 = check((q, empty, empty, whole_k, whole_v), lens + 300)
    _, _, tol, tol_lse = reference(q, pk, pv, k, v, lens, 128 ** -0.5)
    assert bool(((o.double() - o2.double()).abs() <= 2 * tol).all())
    assert bool(((lse.double() - lse2.double()).abs() <= 2 * tol_lse).all())


def test_captured_replayed_and_on_other_streams():
    """Two graphs and eager calls in turn, inputs changed between replays; then calls on two streams at once."""
    import torch

    import neptune_opt_b200 as NB

    one, two = make(4, 8, 2, 1, 128, 600, 300), make(40, 8, 2, 1, 128, 900, 30, seed=1)
    lens = lens_of(300, 20, 0, 111)
    NB.prefix_attention(*one, lens), NB.prefix_attention(*two)
    graphs = []
    for args, n in ((one, lens), (two, None)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = NB.prefix_attention(*args, n, return_lse=True)
        graphs.append((g, out))
    for step in range(3):
        for t in (*one, *two):
            t.mul_(-1.0 if step else 1.0)
        lens.copy_(lens_of(300 - step, 20 + step, step, 111))
        for g, _ in graphs:
            g.replay()
        for (_, got), args, n in zip(graphs, (one, two), (lens, None)):
            want = NB.prefix_attention(*args, n, return_lse=True)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    want = [NB.prefix_attention(*one, lens), NB.prefix_attention(*two)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        got = []
        for s, (args, n) in zip(streams, ((one, lens), (two, None))):
            with torch.cuda.stream(s):
                got.append(NB.prefix_attention(*args, n))
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
