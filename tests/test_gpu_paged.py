"""GPU tests of the paged key/value cache: the append with the rotation on the
way, attention with a window and sinks, and attention behind a shared prefix,
against their definitions in 64 bits."""
import ctypes as C
import math

import numpy as np
import pytest

from tests.paged_testlib import EPS_HALF, Case, torch_dtype
from tests.vox_testlib import vox

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def V():
    return vox()


# ---- append ------------------------------------------------------------------


def rotated(x, pos, theta):
    """The interleaved rotation in 64 bits; x [tokens, heads, dim], pos python ints.
    The angle is reduced by a turn in exact integer arithmetic first."""
    dim = x.shape[-1]
    out = np.empty_like(x)
    for t, a in enumerate(pos):
        for c in range(dim // 2):
            turn = float(theta) ** (-2.0 * c / dim) / (2 * math.pi)
            # 2^60 steps a turn: the position's product with them, modulo a turn
            ang = 2 * math.pi * ((a * int(turn * 2.0 ** 60)) % (1 << 60)) / 2.0 ** 60
            x0, x1 = x[t, :, 2 * c], x[t, :, 2 * c + 1]
            out[t, :, 2 * c] = x0 * math.cos(ang) - x1 * math.sin(ang)
            out[t, :, 2 * c + 1] = x0 * math.sin(ang) + x1 * math.cos(ang)
    return out


APPENDS = [
    # dtype, heads, kv, dim, page, q_len, kv_len, base, layout
    ("bf16", 32, 8, 128, 16, (1,), (1536,), 0, "heads"),
    ("f16", 8, 2, 64, 8, (1, 1, 1), (1, 8, 9), 1000003, "slots"),
    ("f32", 4, 2, 128, 16, (3, 0, 17), (3, 4, 40), 5, "pair"),
    ("bf16", 5, 1, 80, 1, (2, 5), (2, 9), 0, "heads"),
    ("f32", 6, 3, 6, 4, (7, 1), (9, 1), 3, "heads"),       # a row is no multiple of 16 bytes
    ("f16", 2, 2, 256, 64, (33,), (70,), 2 ** 33 + 7, "heads"),  # positions past 32 bits
    ("bf16", 7, 1, 64, 32, tuple([1] * 70), tuple(range(1, 71)), 0, "heads"),
]


@pytest.mark.parametrize("dtype,heads,kv,dim,page,q_len,kv_len,base,layout", APPENDS)
@pytest.mark.parametrize("fused", [False, True])
def test_append_stores_rotated_keys_and_values(V, dtype, heads, kv, dim, page, q_len, kv_len, base, layout, fused):
    c = Case(V, torch, dtype, heads, kv, dim, page, q_len, kv_len, layout=layout, seed=3, poison=False, spare_tokens=2)
    first = torch.tensor([base + 11 * s for s in range(c.n)], dtype=torch.int64, device="cuda")
    batch = V.PagedBatch(c.q_start, c.kv, c.table_dev, c.tokens, max(c.q_len), first_pos=first, status=c.status)
    g = torch.Generator(device="cuda").manual_seed(1)
    if fused:  # views of one projection's rows
        qkv = torch.randn(c.tokens, heads + 2 * kv, dim, generator=g, device="cuda").to(torch_dtype(dtype))
        q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
    else:
        q, k, v = (torch.randn(c.tokens, n, dim, generator=g, device="cuda").to(torch_dtype(dtype))
                   for n in (heads, kv, kv))
    q_in = q.clone()
    theta = 1e6
    before_k, before_v = c.kp.clone(), c.vp.clone()
    got_q = V.paged_append_rope(c.cache, batch, k, v, theta, q=q, q_out=q if fused else None)
    if not fused:
        # rows behind the last sequence are not written: undefined in the new tensor
        got_q = got_q[:sum(q_len)]
    torch.cuda.synchronize()
    assert int(c.status) == 0
    pos = [base + 11 * s + L - n + i for s, (n, L) in enumerate(zip(c.q_len, c.kv_len)) for i in range(n)]
    f64 = lambda t: t.float().cpu().numpy().astype(np.float64)  # noqa: E731
    # a product and a sum of 32 bits and the angle's 2^-24, then one rounding to the type
    u = EPS_HALF[dtype]
    for name, have, src in (("q", got_q, q_in), ("k", None, k)):
        x = f64(src)[:len(pos)]
        want = rotated(x, pos, theta)
        size = np.repeat(np.abs(x[..., 0::2]) + np.abs(x[..., 1::2]), 2, -1)
        tol = u * np.abs(want) + size * 2.0 ** -21
        if name == "k":
            want_k, want_tol = want, tol
        else:
            assert np.all(np.abs(f64(have)[:len(pos)] - want) <= tol)
    if fused:
        assert torch.equal(got_q[sum(q_len):], q_in[sum(q_len):])  # behind the last sequence
    kp, vp, touched = f64(c.kp), c.vp.cpu(), np.zeros(c.kp.shape[:1] + c.kp.shape[2:3], bool)
    at = 0
    for s, (n, L) in enumerate(zip(c.q_len, c.kv_len)):
        for i in range(n):
            page_id, slot = c.table[s, (L - n + i) // page], (L - n + i) % page
            assert np.all(np.abs(kp[page_id, :, slot] - want_k[at]) <= want_tol[at])
            assert torch.equal(vp[page_id, :, slot], v[at].cpu())
            touched[page_id, slot] = True
            at += 1
    same = torch.from_numpy(~touched)[:, None, :, None].expand(c.kp.shape)
    assert torch.equal(c.kp.cpu()[same], before_k.cpu()[same]) and torch.equal(vp[same], before_v.cpu()[same])


def test_append_without_rotation_and_without_queries(V):
    c = Case(V, torch, "f32", 4, 2, 32, 8, (5,), (13,), poison=False)
    k, v = torch.randn(5, 2, 32, device="cuda"), torch.randn(5, 2, 32, device="cuda")
    assert V.paged_append_rope(c.cache, c.batch, k, v, 0.0) is None
    for i in range(5):
        t = 8 + i
        assert torch.equal(c.kp[c.table[0, t // 8], :, t % 8], k[i])
        assert torch.equal(c.vp[c.table[0, t // 8], :, t % 8], v[i])


def test_append_agrees_with_the_frameworks_rotation(V):
    """Same pairs and frequencies as rope_interleaved_inplace (whose 32-bit angle
    is off by up to 2^-24 of the position)."""
    cfg = V.DecoderConfig(dim=8, hidden_dim=16, n_heads=2, n_kv_heads=1, head_dim=4, sliding_window=4,
                          norm_eps=1e-5, rope_theta=1e4)
    c = Case(V, torch, "f32", 4, 4, 64, 16, (6,), (46,), poison=False)
    q = torch.randn(6, 4, 64, device="cuda")
    got = V.paged_append_rope(c.cache, c.batch, q, q, 1e4, q=q).cpu().numpy()
    with V.Context(cfg) as ctx:
        want = V.rope_interleaved_inplace(ctx, q.cpu().numpy().ravel(), 6, 4, 64, 40, 1e4).reshape(6, 4, 64)
    assert np.max(np.abs(got - want)) <= 46 * 2.0 ** -23 * np.abs(want).max() * 2 + 1e-6


def test_append_reports_bad_pages_and_lengths(V):
    c = Case(V, torch, "bf16", 4, 2, 64, 8, (1, 1, 1, 1), (9, 9, 9, 9), poison=False)
    k = torch.randn(4, 2, 64, device="cuda").bfloat16()
    before = c.kp.clone()
    c.table_dev[1, 1] = c.n_pages  # one past the pool
    c.kv[2] = 17                   # beyond the table's two columns
    c.kv[3] = -4
    V.paged_append_rope(c.cache, c.batch, k, k, 0.0)
    assert int(c.status) == V.PAGED_BAD_LENGTH | V.PAGED_BAD_PAGE
    changed = (c.kp != before).flatten(2).any(-1).any(-1).nonzero().flatten().tolist()
    assert changed == [int(c.table[0, 1])]


# ---- attention ---------------------------------------------------------------

# Long and short sequences together
LONG = [
    # dtype, heads, kv, dim, q_len, kv_len, window, sinks
    ("f32", 32, 8, 128, (1,) * 8, (1036, 17, 3000, 0, 1, 900, 16, 257), 0, 0),
    ("bf16", 8, 8, 128, (1, 0, 2, 1, 1) * 3, (1, 5, 2000, 333, 48) * 3, 700, 5),
    ("f16", 16, 8, 64, (2, 1, 8) * 20, (900, 64, 8) * 20, 0, 0),
    ("bf16", 8, 8, 128, (1,) * 100, (1, 2, 3, 4) * 24 + (800, 1, 1, 0), 0, 0),
    ("bf16", 16, 8, 128, (1,) * 3, (5000, 16, 1), 4500, 40),
]


@pytest.mark.parametrize("dtype,heads,kv,dim,q_len,kv_len,window,sinks", LONG)
@pytest.mark.parametrize("prefix", [0, 30])
def test_decode_long_and_short(V, dtype, heads, kv, dim, q_len, kv_len, window, sinks, prefix):
    c = Case(V, torch, dtype, heads, kv, dim, 16, q_len, kv_len, window, sinks, prefix=prefix, seed=25, spare_tokens=2)
    out = torch.full_like(c.q, 3.0)
    c.run(out=out)
    assert bool((out[sum(q_len):] == 3.0).all())
    c.check(out)
    assert int(c.status) == 0
    again = torch.full_like(c.q, 3.0)
    c.run(out=again)
    assert torch.equal(out, again)


def test_bad_sequences_among_long_ones(V):
    c = Case(V, torch, "bf16", 8, 8, 128, 16, (1,) * 8, (900, 1600, 30, 700, 1, 1500, 44, 90), seed=26, poison=False)
    want = c.run()
    c.kv[1] = 1601
    c.kv[4] = -1
    c.table_dev[5, 3] = -2
    out = torch.full_like(want, 9.0)
    c.run(out=out)
    assert int(c.status) == V.PAGED_BAD_LENGTH | V.PAGED_BAD_PAGE
    for s in range(8):
        if s in (1, 4):
            assert bool((out[s] == 9.0).all())
        elif s != 5:
            assert torch.equal(out[s], want[s])
    c.q_start.fill_(0)  # no tokens at all
    out.fill_(9.0)
    c.run(out=out)
    assert bool((out == 9.0).all())


SHAPES = [  # heads, kv_heads, dim
    (32, 8, 128), (8, 1, 64), (4, 4, 128), (10, 2, 64), (7, 1, 128), (6, 2, 80), (2, 1, 256), (3, 3, 6),
]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("heads,kv,dim", SHAPES)
def test_decode_ragged(V, dtype, heads, kv, dim):
    c = Case(V, torch, dtype, heads, kv, dim, 16, (1, 1, 1, 0, 1, 1, 1), (1, 2, 16, 5, 17, 130, 333), seed=1)
    c.check(c.run())
    assert int(c.status) == 0


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("page", [1, 4, 8, 16, 64, 128, 256])
@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 0), (64, 4), (33, 70), (1, 1), (1000, 3)])
def test_decode_window_and_sinks(V, dtype, page, window, sinks):
    c = Case(V, torch, dtype, 8, 2, 64, page, (1, 1, 2, 1), (7, 300, 401, 129), window, sinks, seed=page)
    c.check(c.run())
    assert int(c.status) == 0


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("heads,kv,dim", SHAPES)
@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 5)])
def test_prefill_ragged(V, dtype, heads, kv, dim, window, sinks):
    c = Case(V, torch, dtype, heads, kv, dim, 32, (3, 100, 0, 257, 1), (3, 100, 7, 290, 65), window, sinks, seed=2)
    c.check(c.run())
    assert int(c.status) == 0


@pytest.mark.parametrize("dtype,dim", [("bf16", 64), ("f16", 128)])
@pytest.mark.parametrize("window,sinks,longest", [(0, 0, 1500), (600, 4, 1500)])
def test_a_last_wave_of_few_tiles(V, dtype, dim, window, sinks, longest):
    """152 tiles of 256 rows: 148 as they are, the last 4 in parts."""
    q_len = tuple(65 - (i % 3 == 1) for i in range(19))
    kv_len = tuple(longest - 70 * i for i in range(19))
    c = Case(V, torch, dtype, 16, 4, dim, 16, q_len, kv_len, window, sinks, seed=28, spare_tokens=5)
    c.v[18][kv_len[18] - 1, 0, 3] = math.nan  # seen by the last token alone, in a split tile or not
    c.vp[c.table[18, (kv_len[18] - 1) // 16], 0, (kv_len[18] - 1) % 16, 3] = math.nan
    c.v[0][longest - 1, 1, 5] = math.inf
    c.vp[c.table[0, (longest - 1) // 16], 1, (longest - 1) % 16, 5] = math.inf
    out = torch.full_like(c.q, 3.0)
    c.run(out=out)
    assert bool((out[sum(q_len):] == 3.0).all()) and int(c.status) == 0
    want, tol = c.expected()
    got = out.float().cpu().numpy()[:sum(q_len)]
    want, tol = want[:sum(q_len)], tol[:sum(q_len)]
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(np.isinf(got), np.isinf(want))
    ok = np.isfinite(want)
    assert np.all(np.abs(got[ok] - want[ok]) <= tol[ok])
    # the same plan for queries that are not on 16-byte boundaries
    odd = torch.empty(c.q.numel() + 1, device="cuda", dtype=c.q.dtype)[1:].view(c.q.shape)
    odd.copy_(c.q)
    got = c.run(q=odd).float().cpu().numpy()[:sum(q_len)]
    assert np.all(np.abs(got[ok] - want[ok]) <= tol[ok])


def test_windows_beyond_every_length(V):
    for dtype, q_len in (("bf16", (1, 40)), ("f32", (3, 1))):
        c = Case(V, torch, dtype, 8, 2, 64, 16, q_len, (90, 70), seed=29)
        for window in (91, 1 << 31, (1 << 64) - 1):
            got = V.paged_attention(c.cache, c.batch, c.q, sliding_window=window, n_sinks=(1 << 64) - 1)
            c.check(got)


@pytest.mark.parametrize("layout", ["heads", "slots", "pair"])
@pytest.mark.parametrize("dim,page", [(128, 16), (64, 128), (64, 8)])
@pytest.mark.parametrize("q_len,kv_len", [((1, 1), (77, 300)), ((120, 65), (400, 65))])
def test_pool_layouts(V, layout, dim, page, q_len, kv_len):
    c = Case(V, torch, "bf16", 8, 2, dim, page, q_len, kv_len, 60, 3, layout=layout, seed=5)
    c.check(c.run())


def test_strided_queries_and_outputs(V):
    for q_len, kv_len in (((1, 1), (40, 90)), ((70, 130), (70, 200))):
        c = Case(V, torch, "bf16", 8, 2, 128, 16, q_len, kv_len, seed=6)
        wide = torch.full((c.tokens, 11, 128), 7.0, device="cuda", dtype=torch.bfloat16)
        wide[:, 2:10] = c.q
        out = torch.full((8, c.tokens, 136), 5.0, device="cuda", dtype=torch.bfloat16)
        view = out[:, :, :128].transpose(0, 1)
        assert c.run(q=wide[:, 2:10], out=view) is view
        c.check(view.contiguous())
        assert bool((out[:, :, 128:] == 5.0).all())
        # odd offsets: rows that do not start on a 16-byte boundary
        odd = torch.empty(c.tokens * 8 * 128 + 1, device="cuda", dtype=torch.bfloat16)[1:].view(c.tokens, 8, 128)
        odd.copy_(c.q)
        c.check(c.run(q=odd))


def test_rows_behind_the_last_sequence_stay(V):
    for q_len, kv_len, prefix in (((1, 1), (5, 90), 0), ((70, 3), (70, 200), 0), ((1, 2), (5, 9), 100)):
        c = Case(V, torch, "bf16", 8, 2, 64, 16, q_len, kv_len, prefix=prefix, spare_tokens=5, seed=7)
        out = torch.full((c.tokens, 8, 64), 3.0, device="cuda", dtype=torch.bfloat16)
        c.run(out=out)
        assert bool((out[sum(q_len):] == 3.0).all())
        c.check(torch.cat((out[:sum(q_len)], out[sum(q_len):] * math.nan)))


def test_more_queries_than_cached_tokens(V):
    for dtype in ("bf16", "f32"):
        c = Case(V, torch, dtype, 8, 2, 64, 16, (4, 300, 1), (2, 200, 0), seed=8)
        got = c.run()
        c.check(got)
        assert bool((got[:2] == 0).all()) and bool((got[-1] == 0).all())


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("n", [5, 40, 300])
def test_nan_and_infinity_reach_only_who_sees_them(V, dtype, n):
    """A NaN value at the last token, an infinite one in the middle: the tokens
    before them, in the same tiles, and those past the window stay finite."""
    c = Case(V, torch, dtype, 4, 2, 64, 16, (n,), (n + 30,), window=20, sinks=2, seed=9)
    L = n + 30
    for t, x in ((L - 1, math.nan), (31, math.inf)):
        c.v[0][t, 0, 3] = x
        c.vp[c.table[0, t // 16], 0, t % 16, 3] = x
    c.k[0][L - 2, 1] = math.nan
    c.kp[c.table[0, (L - 2) // 16], 1, (L - 2) % 16] = math.nan
    got = c.run().float().cpu().numpy()
    want, tol = c.expected()
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(np.isinf(got), np.isinf(want))
    ok = np.isfinite(want)
    assert ok.any() and np.all(np.abs(got[ok] - want[ok]) <= tol[ok])


def test_scale_and_large_scores(V):
    c = Case(V, torch, "bf16", 8, 2, 64, 16, (1, 90), (100, 90), seed=10, q_scale=30.0)
    c.check(c.run())
    c = Case(V, torch, "f32", 8, 2, 64, 16, (1, 90), (100, 90), seed=10)
    c.check(c.run(scale=0.7), scale=0.7)


def test_bad_pages_and_lengths_are_reported(V):
    for q_len in ((1, 1, 1, 1), (80, 80, 80, 80)):
        c = Case(V, torch, "bf16", 8, 2, 64, 16, q_len, (90, 95, 90, 96), seed=11, poison=False)
        want = c.run()
        c.table_dev[1, 2] = c.n_pages + 5
        c.kv[2] = 97  # beyond the table
        out = torch.full_like(want, 9.0)
        c.run(out=out)
        assert int(c.status) == V.PAGED_BAD_LENGTH | V.PAGED_BAD_PAGE
        n = q_len[0]
        assert torch.equal(out[:n], want[:n]) and torch.equal(out[3 * n:], want[3 * n:])
        assert bool(torch.isfinite(out).all()) and bool((out[2 * n:3 * n] == 9.0).all())
        # a bad page that no token needs is not looked at
        d = Case(V, torch, "bf16", 8, 2, 64, 16, (1,), (95,), window=20, seed=11)
        d.table_dev[0, 1] = -77
        d.check(d.run())
        assert int(d.status) == 0


def test_offsets_past_32_bits(V):
    """A pool of over 2^32 elements, its first and last pages in use."""
    pages, hd = 33000, 128
    k = torch.empty(pages, 8, 128, hd, dtype=torch.bfloat16, device="cuda")
    v = torch.empty_like(k)
    assert k.numel() > 2 ** 32
    c = Case(V, torch, "bf16", 32, 8, hd, 128, (1, 3), (200, 250), seed=12)
    big = {int(x): (pages - 1 - i if i % 2 else i) for i, x in enumerate(sorted(set(c.table[c.table >= 0].tolist())))}
    for src, dst in big.items():
        k[dst], v[dst] = c.kp[src], c.vp[src]
    table = torch.tensor([[big.get(int(x), -1) for x in row] for row in c.table], dtype=torch.int32, device="cuda")
    cache = V.PagedKvCache(k, v)
    batch = V.PagedBatch(c.q_start, c.kv, table, c.tokens, 3)
    c.check(V.paged_attention(cache, batch, c.q))
    new = torch.randn(c.tokens, 8, hd, device="cuda").bfloat16()
    V.paged_append_rope(cache, batch, new, new, 0.0)
    assert torch.equal(k[int(table[0, 199 // 128]), :, 199 % 128], new[0])


# ---- shared prefix -------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("heads,kv,dim", SHAPES)
@pytest.mark.parametrize("prefix,q_len,kv_len", [
    (1, (1,), (1,)), (100, (1, 1, 1), (1, 20, 7)), (300, (1, 3, 0, 2, 4), (40, 3, 9, 2, 17)),
    (65, tuple([1] * 40), tuple(range(1, 41))),
])
def test_prefix(V, dtype, heads, kv, dim, prefix, q_len, kv_len):
    c = Case(V, torch, dtype, heads, kv, dim, 16, q_len, kv_len, prefix=prefix, seed=13)
    c.check(c.run())
    assert int(c.status) == 0


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("window,sinks", [(30, 0), (30, 4), (200, 150), (5, 400), (290, 3)])
def test_prefix_window_and_sinks(V, dtype, window, sinks):
    c = Case(V, torch, dtype, 8, 2, 128, 32, (1, 1, 4, 2) + (1,) * 30, (1, 90, 40, 2) + (25,) * 30, window, sinks,
             prefix=280, seed=14)
    c.check(c.run())
    assert int(c.status) == 0


# Long enough, or with enough rows, to be computed once for all sequences (a short
# prefix is the first part of every sequence's keys).
SHARED = [
    # heads, kv, dim, prefix, q_len, kv_len
    (8, 2, 64, 2100, (1,) * 40, tuple(range(1, 41))),
    (8, 2, 128, 1111, (1, 0, 2, 1) * 10, (30, 4, 9, 1) * 10),
    (8, 1, 128, 130, (5, 1, 4), (40, 1, 3)),       # 40 rows a sequence: tcgen05 for its own keys too
    (4, 4, 128, 3000, (1,) * 12, (7,) * 12),       # 12 rows for the prefix
    (12, 2, 80, 1200, (1, 2) * 30, (3, 20) * 30),  # CUDA cores
]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("heads,kv,dim,prefix,q_len,kv_len", SHARED)
@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 3), (900, 1000)])
def test_shared_prefix(V, dtype, heads, kv, dim, prefix, q_len, kv_len, window, sinks):
    c = Case(V, torch, dtype, heads, kv, dim, 16, q_len, kv_len, window, sinks, prefix=prefix, seed=23, spare_tokens=3)
    out = torch.full_like(c.q, 3.0)
    c.run(out=out)
    assert bool((out[sum(q_len):] == 3.0).all())
    c.check(out)
    assert int(c.status) == 0


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("prefix,page", [(1, 256), (300, 64), (128, 128)])
def test_prefix_that_no_window_reaches(V, dtype, prefix, page):
    """Its pages (-1 in the list) are not looked at."""
    c = Case(V, torch, dtype, 14, 2, 128, page, (64, 50), (155, 97), 5, 0, prefix=prefix, seed=27)
    assert (c.pre == -1).all()
    c.check(c.run())
    assert int(c.status) == 0


def test_bad_shared_prefix_is_reported(V):
    c = Case(V, torch, "bf16", 8, 2, 128, 16, (1,) * 40, (5,) * 40, prefix=1200, seed=24)
    want = c.run()
    for n in (-1, 1201):
        c.pre_len.fill_(n)
        c.status.zero_()
        out = torch.full_like(want, 4.0)
        c.run(out=out)
        assert int(c.status) == V.PAGED_BAD_LENGTH and bool((out == 4.0).all())
    c.pre_len.fill_(1200)
    c.status.zero_()
    c.pre_dev[7] = 1 << 30
    assert bool(torch.isfinite(c.run()).all()) and int(c.status) == V.PAGED_BAD_PAGE


def test_prefix_equals_attention_on_whole_sequences(V):
    """The same tokens as one paged sequence each: equal up to the rounding of
    weights and results (two of each)."""
    c = Case(V, torch, "f16", 8, 2, 64, 16, (1, 2, 1), (5, 20, 33), prefix=64, seed=15)
    got = c.run()
    table = torch.cat((c.pre_dev[None].expand(3, -1), c.table_dev), 1).contiguous()
    batch = V.PagedBatch(c.q_start, c.kv + 64, table, c.tokens, 2)
    whole = V.paged_attention(c.cache, batch, c.q)
    want, tol = c.expected()
    assert np.all(np.abs((got - whole).float().cpu().numpy()) <= 2 * tol)


def test_bad_prefix_is_reported(V):
    c = Case(V, torch, "bf16", 8, 2, 64, 16, (1, 2), (5, 20), prefix=64, seed=16)
    want = c.run()
    for n in (-1, 65):
        c.pre_len.fill_(n)
        c.status.zero_()
        out = torch.full_like(want, 4.0)
        c.run(out=out)
        assert int(c.status) == V.PAGED_BAD_LENGTH and bool((out == 4.0).all())
    c.pre_len.fill_(64)
    c.status.zero_()
    c.pre_dev[1] = -9
    assert bool(torch.isfinite(c.run()).all()) and int(c.status) == V.PAGED_BAD_PAGE


# ---- used together, graphs, streams ---------------------------------------------


def test_graph_replays_follow_the_device_arrays(V):
    """append + attention captured once for bounds, replayed as the sequences grow."""
    c = Case(V, torch, "bf16", 8, 2, 128, 16, (1, 1, 1), (200, 64, 150), seed=17, poison=False)
    batch = V.PagedBatch(c.q_start, c.kv, c.table_dev, 3, 1, status=c.status)
    k, v, q = (torch.randn(3, n, 128, device="cuda").bfloat16() for n in (2, 2, 8))
    full = c.kv.clone()

    def step():
        qr = V.paged_append_rope(c.cache, batch, k, v, 1e4, q=q)
        return V.paged_attention(c.cache, batch, qr, sliding_window=100, n_sinks=4)

    c.kv.copy_(full - 3)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for back in (3, 2, 1, 0):
        c.kv.copy_(full - back)
        for x in (k, v, q):
            x.normal_()
        kp, vp = c.kp.clone(), c.vp.clone()
        want = step()
        c.kp.copy_(kp)
        c.vp.copy_(vp)
        out.zero_()
        graph.replay()
        assert torch.equal(out, want)
    assert int(c.status) == 0


def test_two_graphs_and_two_streams_do_not_share_scratch(V):
    cases = [Case(V, torch, "bf16", 8, 2, 128, 16, (1,), (900 + 40 * i,), seed=18 + i) for i in range(2)]
    cases += [Case(V, torch, "bf16", 8, 2, 128, 16, (1,) * 9, (9,) * 9, prefix=3700 + i, seed=28 + i) for i in range(2)]
    want = [c.run() for c in cases]
    graphs, outs = [], []
    for c in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(c.run())
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert torch.equal(o, w)
    for _ in range(20):
        got = []
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                got.append(c.run())
        torch.cuda.synchronize()
        for o, w in zip(got, want):
            assert torch.equal(o, w)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_results_do_not_depend_on_the_run(V, dtype):
    for q_len, kv_len, prefix in (((1, 1), (3000, 17), 0), ((200,), (1300,), 0), ((1,) * 20, (30,) * 20, 1000),
                                 ((1,) * 40, (30,) * 40, 2000)):
        c = Case(V, torch, dtype, 8, 2, 128, 16, q_len, kv_len, prefix=prefix, seed=19, poison=False)
        first = c.run()
        for _ in range(5):
            assert torch.equal(c.run(), first)


def test_decoding_with_the_cache(V):
    """A prompt appended and attended to in ragged chunks, then tokens one by
    one, then hypotheses behind it: every step equals attention over all tokens
    so far in 64 bits."""
    heads, kv, dim, page, theta = 8, 2, 64, 16, 1e4
    td = torch.bfloat16
    g = torch.Generator(device="cuda").manual_seed(20)
    kp = torch.full((40, kv, page, dim), math.nan, device="cuda", dtype=td)
    vp = torch.full_like(kp, math.nan)
    cache = V.PagedKvCache(kp, vp)
    table = torch.arange(30, dtype=torch.int32, device="cuda").flip(0)[None].contiguous()
    i32 = dict(dtype=torch.int32, device="cuda")
    keys, values, n = [], [], 0

    def reference(q, k, v, first):
        q, k, v = (t.float().cpu().numpy().astype(np.float64) for t in (q, k, v))
        out = np.zeros_like(q)
        for i in range(q.shape[0]):
            m = first + i + 1
            kk, vv = (np.repeat(t[:m], heads // kv, 1) for t in (k, v))
            s = np.einsum("hd,jhd->hj", q[i], kk) / math.sqrt(dim)
            w = np.exp(s - s.max(-1, keepdims=True))
            out[i] = np.einsum("hj,jhd->hd", w / w.sum(-1, keepdims=True), vv)
        return out

    def stored(a, b):
        at = torch.arange(a, b, device="cuda")
        return kp[table[0, at // page].long(), :, at % page], vp[table[0, at // page].long(), :, at % page]

    for m in (100, 37, 1, 1, 1):
        q, k, v = (torch.randn(m, h, dim, generator=g, device="cuda").to(td) for h in (heads, kv, kv))
        n += m
        batch = V.PagedBatch(torch.tensor([0, m], **i32), torch.tensor([n], **i32), table, m, m)
        qr = V.paged_append_rope(cache, batch, k, v, theta, q=q)
        out = V.paged_attention(cache, batch, qr)
        kk, vv = stored(0, n)
        assert torch.equal(vv[n - m:], v)
        keys.append(k)
        # |values| below 5, weights and results each rounded to bf16
        want = reference(qr, kk, vv, n - m)
        assert np.max(np.abs(out.float().cpu().numpy() - want)) <= 3 * 5 * 2.0 ** -8
    # three hypotheses of two tokens each behind it, in pages of their own
    q, k, v = (torch.randn(6, h, dim, generator=g, device="cuda").to(td) for h in (heads, kv, kv))
    own = torch.tensor([[31], [33], [38]], **i32)
    batch = V.PagedBatch(torch.tensor([0, 2, 4, 6], **i32), torch.tensor([2, 2, 2], **i32), own, 6, 2,
                         first_pos=torch.full((3,), n, dtype=torch.int64, device="cuda"))
    qr = V.paged_append_rope(cache, batch, k, v, theta, q=q)
    out = V.paged_prefix_attention(cache, batch, table[0], torch.tensor([n], **i32), 160, qr)
    kk, vv = stored(0, n)
    for h in range(3):
        mine = (t[int(own[h, 0]), :, :2].transpose(0, 1) for t in (kp, vp))
        ck, cv = (torch.cat(x) for x in zip((kk, vv), mine))
        want = reference(qr[2 * h:2 * h + 2], ck, cv, n)
        assert np.max(np.abs(out[2 * h:2 * h + 2].float().cpu().numpy() - want)) <= 3 * 5 * 2.0 ** -8


def test_empty_batches(V):
    c = Case(V, torch, "bf16", 8, 2, 64, 16, (0, 0), (5, 0), seed=21)
    assert c.run(q=torch.empty(0, 8, 64, device="cuda", dtype=torch.bfloat16)).shape == (0, 8, 64)
    out = V.paged_append_rope(c.cache, c.batch, torch.empty(0, 2, 64, device="cuda", dtype=torch.bfloat16),
                              torch.empty(0, 2, 64, device="cuda", dtype=torch.bfloat16), 1e4)
    assert out is None


def test_workspace_is_checked(V):
    c = Case(V, torch, "bf16", 8, 2, 64, 16, (1,) * 60, (5, 9) * 30, prefix=1100, seed=22, max_kv=16)
    L = V.lib()
    pre = V.PagedPrefixDesc(c.pre_dev.data_ptr(), c.pre_len.data_ptr(), len(c.pre), 1100)
    n = C.c_size_t()
    assert L.vox_paged_prefix_attention_workspace(c.cache._ref, c.batch._ref, C.byref(pre), 8, 0, 0, C.byref(n)) == 0
    assert n.value > 0
    ws = torch.empty(n.value + 256, dtype=torch.uint8, device="cuda")
    out = torch.empty_like(c.q)
    rows = [V.Rows(t.data_ptr(), 0, 0) for t in (c.q, out)]
    call = lambda p, m: L.vox_paged_prefix_attention(c.cache._ref, c.batch._ref, C.byref(pre), C.byref(rows[0]), 8, 0,  # noqa: E731
                                                     0, 0.0, C.byref(rows[1]), p, m, None)
    assert call(ws.data_ptr(), n.value - 1) == V.ERR_INVALID_ARG
    assert call(ws.data_ptr() + 64, n.value) == V.ERR_INVALID_ARG
    assert call(None, n.value) == V.ERR_INVALID_ARG
    torch.cuda.synchronize()
    assert call(ws.data_ptr(), n.value) == 0
    torch.cuda.synchronize()
    c.check(out)
