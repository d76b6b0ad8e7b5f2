"""GPU tests of the paged-cache attention where single keys outweigh all others,
where calls share what they should not, and where arguments are at their limits."""
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


def store(c):
    """Puts a case's changed keys and values (c.k, c.v, c.pk, c.pv) into its pool."""
    for s in range(c.n):
        t = np.arange(c.kv_len[s])
        page = torch.from_numpy(c.table[s, t // c.page].astype(np.int64))
        for pool, x in ((c.kp, c.k[s]), (c.vp, c.v[s])):
            pool[page.cuda(), :, torch.from_numpy(t % c.page).cuda()] = x.cuda()
    t = np.arange(c.prefix)
    page = torch.from_numpy(c.pre[t // c.page].astype(np.int64))
    for pool, x in ((c.kp, c.pk), (c.vp, c.pv)):
        pool[page.cuda(), :, torch.from_numpy(t % c.page).cuda()] = x.cuda()


def dominated(V, dtype, gap, spread, sinks, **kw):
    """Every query scores about `gap` nats more on the keys `sinks` (of the prefix
    where there is one) than on any other, and their values are 0: a result is what
    the others add.  `spread` scales the others' keys; their values are positive."""
    c = Case(V, torch, dtype, poison=False, **kw)
    q = c.q_host
    q[..., 0] = 8.0
    q[..., 1:] *= 0.5
    c.q = q.cuda()
    for k, v in [(c.pk, c.pv)] + list(zip(c.k, c.v)):
        k *= spread
        k[..., 0] = 0.0
        v.abs_()
    k, v = (c.pk, c.pv) if c.prefix else (c.k[0], c.v[0])
    for j in sinks:
        k[j] = 0.0
        k[j, :, 0] = gap * math.sqrt(c.dim) / 8.0
        v[j] = 0.0
    store(c)
    return c


def check_dominated(c, got):
    """Beyond Case.expected's tolerance: a result below f16's normal range is
    rounded by up to 2^-25, and the weights of the keys beside a dominating one may
    be rounded by up to 2^-33 of that one's each, 64 of them at most in a step of
    keys that share a scale (2^-40 of 8192 keys come to less): 2^-27 of a value."""
    want, tol = c.expected()
    got = got.detach().cpu().double().numpy()
    n = sum(c.q_len)
    top = max(float(x.float().abs().max()) for x in c.v + ([c.pv] if c.prefix else []) if x.numel())
    if c.dtype == "f16":
        tol = tol + 2.0 ** -25 + 2.0 ** -27 * top
    off = np.abs(got - want)[:n] - tol[:n]
    assert np.all(off <= 0), f"{off.max():.3e} over the tolerance; relative {np.max(np.abs(got / want - 1)[:n]):.3e}"


DOMINATED = [
    # heads, kv, dim, q_len, kv_len, prefix, sinks
    (4, 1, 128, (1,), (8192,), 0, (0,)),                    # one stream's decode
    (8, 2, 64, (1, 2, 1), (6000, 40, 700), 0, (0, 3)),      # few rows
    (4, 1, 128, (20,), (5000,), 0, (0,)),                   # tcgen05 tiles
    (4, 1, 64, (40, 3), (4000, 70), 0, (1500, 0)),          # the same, the dominating key in the middle too
    (8, 2, 128, (1,) * 12, (30,) * 12, 4000, (0,)),         # a shared prefix, joined with the sequences' own
    (4, 1, 64, (20,), (40,), 0, (1,)),                      # few keys
]


@pytest.mark.parametrize("dtype,gap", [("f16", 10.0), ("f16", 14.0), ("f16", 18.0), ("bf16", 16.0), ("f32", 16.0)])
@pytest.mark.parametrize("spread", [0.0, 1.0])
@pytest.mark.parametrize("heads,kv,dim,q_len,kv_len,prefix,sinks", DOMINATED)
def test_keys_beside_a_dominating_one(V, dtype, spread, gap, heads, kv, dim, q_len, kv_len, prefix, sinks):
    c = dominated(V, dtype, gap, spread, sinks, heads=heads, kv_heads=kv, dim=dim, q_len=q_len, kv_len=kv_len,
                  prefix=prefix, seed=31)
    check_dominated(c, c.run())
    assert int(c.status) == 0


@pytest.mark.parametrize("q_len", [(1,), (20,)])
def test_dominating_keys_on_several_levels(V, q_len):
    """Scores that rise and fall by up to 55 nats every few hundred keys: the
    results follow the highest level whatever came before it, and what adds to them
    at one level is not lost beside a key of value 0 at a higher one."""
    c = dominated(V, "f16", 15.0, 1.0, (0, 64, 2000, 2001), heads=4, kv_heads=1, dim=128, q_len=q_len, kv_len=(4000,),
                  seed=32)
    for a, b, level in ((300, 700, -40.0), (1000, 1100, 3.0), (2500, 3000, -20.0)):
        c.k[0][a:b, :, 0] = level * math.sqrt(c.dim) / 8.0
    store(c)
    check_dominated(c, c.run())


EXPIRED = [
    # dtype, heads, kv, dim, page, q_len, kv_len, prefix
    ("bf16", 8, 2, 128, 16, (40,), (1500,), 0),        # the ring of K and V tiles goes round; keys end inside a page
    ("f16", 4, 1, 64, 64, (70, 9), (900, 70), 0),      # two tiles of a sequence, one with a single row group
    ("bf16", 8, 1, 128, 128, (20, 300), (100, 300), 0),
    ("f16", 8, 2, 128, 16, (1,) * 40, (5,) * 40, 4000),  # parts of a prefix, then the merge
]


@pytest.mark.parametrize("dtype,heads,kv,dim,page,q_len,kv_len,prefix", EXPIRED)
def test_expired_waits_are_reported(V, dtype, heads, kv, dim, page, q_len, kv_len, prefix):
    """Waits that give up after a few polls while all arrives, and waits for tiles
    that never come: the call ends, says so, and the next one is right."""
    c = Case(V, torch, dtype, heads, kv, dim, page, q_len, kv_len, prefix=prefix, seed=33)
    want = c.run()
    limit = V.lib().vox_paged_test_waits
    limit.restype = None
    try:
        for polls, units in ((1, -1), (2, -1), (5, -1), (1, 0), (20, 1), (20, 2), (20, 5)):
            limit(polls, units)
            for _ in range(3):
                c.status.zero_()
                out = c.run()
                torch.cuda.synchronize()
                # (every case has CTAs with 4 blocks of keys or more, or with one: 2 tiles)
                assert int(c.status) in ((V.PAGED_TIMEOUT,) if units in (0, 1) else (0, V.PAGED_TIMEOUT))
                if int(c.status) == 0:
                    assert torch.equal(out, want)
    finally:
        limit(-1, -1)
    c.status.zero_()
    assert torch.equal(c.run(), want) and int(c.status) == 0


def test_a_call_after_a_failed_allocation(V):
    """The failure is the failed call's alone."""
    cfg = V.DecoderConfig(dim=8, hidden_dim=16, n_heads=2, n_kv_heads=1, head_dim=4, sliding_window=4, norm_eps=1e-5,
                          rope_theta=1e4)
    c = Case(V, torch, "bf16", 8, 2, 64, 16, (1, 2), (40, 90), seed=34)
    with V.Context(cfg) as ctx:
        with pytest.raises(V.VoxError) as e:
            V.RollingKvCache(ctx, 4, 8, 128, 1 << 29)  # 8 TB and more
        assert e.value.code == V.ERR_OOM
        c.check(c.run())


def test_a_batch_serves_pools_of_different_page_sizes(V):
    """Each call has the bound of its own pool, whatever calls another thread makes
    with the same batch in between."""
    c = Case(V, torch, "bf16", 8, 2, 64, 16, (1, 2), (70, 90), seed=35)
    small = Case(V, torch, "bf16", 8, 2, 64, 8, (1,), (5,), seed=36)
    mine = C.cast(c.batch._for(c.cache), C.POINTER(V.PagedBatchDesc)).contents
    other = C.cast(c.batch._for(small.cache), C.POINTER(V.PagedBatchDesc)).contents
    width = c.table_dev.shape[1]
    assert (mine.max_kv_len, other.max_kv_len) == (16 * width, 8 * width)
    c.check(c.run())
    assert int(c.status) == 0


def test_a_batch_tells_what_its_calls_met(V):
    """Without a status tensor of the caller's too."""
    c = Case(V, torch, "bf16", 8, 2, 64, 16, (1, 40), (70, 90), seed=37, poison=False)
    batch = V.PagedBatch(c.q_start, c.kv, c.table_dev, c.tokens, 40)
    V.paged_attention(c.cache, batch, c.q)
    batch.check()
    c.kv[0] = -1
    V.paged_attention(c.cache, batch, c.q)
    with pytest.raises(V.VoxError, match="lengths") as e:
        batch.check()
    assert e.value.code == V.ERR_RANGE and "page ids" not in e.value.message
    batch.check()  # cleared
    c.kv[0] = 70
    c.table_dev[1, 0] = c.n_pages
    k = torch.zeros(c.tokens, 2, 64, device="cuda", dtype=torch.bfloat16)
    c.kv[1] = 40
    V.paged_append_rope(c.cache, batch, k, k, 0.0)
    with pytest.raises(V.VoxError, match="page ids"):
        batch.check()
    mine = V.PagedBatch(c.q_start, c.kv, c.table_dev, c.tokens, 40, status=c.status)
    V.paged_attention(c.cache, mine, c.q)
    with pytest.raises(V.VoxError, match="page ids"):
        mine.check()
    assert int(c.status) == 0


def test_a_batch_that_lives_on_keeps_little(V):
    c = Case(V, torch, "bf16", 8, 2, 64, 16, (1, 2), (70, 90), seed=38, poison=False)
    want = V.paged_attention(c.cache, c.batch, c.q, sliding_window=1000)
    for n in range(300):
        got = V.paged_attention(c.cache, c.batch, c.q, sliding_window=1000 + n, n_sinks=n)
        assert torch.equal(got, want)
    assert len(c.batch._workspace_bytes) <= 64


@pytest.mark.parametrize("n", [5, 70])
@pytest.mark.parametrize("what", ["cached", "order"])
def test_append_reports_bad_sequences_without_tokens(V, n, what):
    """As the attention does: also those that no token of the call belongs to."""
    q_len = [1] * n
    q_len[3] = 0
    c = Case(V, torch, "bf16", 4, 2, 64, 8, q_len, [9] * n, seed=39, poison=False)
    if what == "cached":
        c.kv[3] = -4
    else:
        c.q_start[-1] = 0  # the last sequence ends before it begins
    k = torch.zeros(c.tokens, 2, 64, device="cuda", dtype=torch.bfloat16)
    V.paged_append_rope(c.cache, c.batch, k, k, 0.0)
    assert int(c.status) == V.PAGED_BAD_LENGTH
    c.status.zero_()
    V.paged_attention(c.cache, c.batch, torch.zeros(c.tokens, 4, 64, device="cuda", dtype=torch.bfloat16))
    assert int(c.status) == V.PAGED_BAD_LENGTH


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("heads,kv,dim,seqs,tokens", [(8, 2, 128, 3, 1185), (32, 8, 128, 40, 1300), (4, 1, 64, 1, 2400),
                                                      (2, 2, 256, 1201, 1201)])
def test_append_of_many_tokens(V, dtype, heads, kv, dim, seqs, tokens):
    """From 1184 tokens on a block of threads takes two; the last one here has one
    or two, and rows behind the last sequence stay."""
    page, theta, base, spare = 16, 1e6, 70001, 2 if tokens % 2 == 0 else 3
    cut = np.linspace(0, tokens, seqs + 1).astype(int)
    q_len = np.diff(cut)
    kv_len = q_len + np.arange(seqs) % 7
    width = -(-int(kv_len.max()) // page)
    rng = np.random.default_rng(40)
    order = rng.permutation(seqs * width + 2).astype(np.int32)
    table = order[:seqs * width].reshape(seqs, width)
    shape = (len(order), kv, page, dim)
    g = torch.Generator(device="cuda").manual_seed(41)
    td = torch_dtype(dtype)
    kp, vp = (torch.randn(shape, generator=g, device="cuda").to(td) for _ in range(2))
    before = kp.clone(), vp.clone()
    qkv = torch.randn(tokens + spare, heads + 2 * kv, dim, generator=g, device="cuda").to(td)
    first = qkv.clone()
    dev = dict(device="cuda")
    batch = V.PagedBatch(torch.from_numpy(cut.astype(np.int32)).to(**dev), torch.from_numpy(kv_len.astype(np.int32)).to(**dev),
                         torch.from_numpy(table).to(**dev), tokens + spare, int(q_len.max()),
                         first_pos=torch.full((seqs,), base, dtype=torch.int64, device="cuda"))
    q = qkv[:, :heads]
    assert V.paged_append_rope(V.PagedKvCache(kp, vp), batch, qkv[:, heads:heads + kv], qkv[:, heads + kv:], theta, q=q,
                               q_out=q) is q
    batch.check()
    assert torch.equal(qkv[tokens:], first[tokens:]) and torch.equal(qkv[:, heads:], first[:, heads:])
    seq = np.repeat(np.arange(seqs), q_len)
    index = kv_len[seq] - q_len[seq] + np.arange(tokens) - cut[seq]
    ang = (base + index)[:, None] * theta ** (-np.arange(0, dim, 2) / dim)
    cos, sin = (torch.from_numpy(f(ang)).cuda()[:, None] for f in (np.cos, np.sin))

    def check(got, x):
        x0, x1 = x[..., 0::2].double(), x[..., 1::2].double()
        want = torch.stack((x0 * cos - x1 * sin, x0 * sin + x1 * cos), -1).flatten(-2)
        size = (x0.abs() + x1.abs()).repeat_interleave(2, -1)
        # a product and a sum of 32 bits and the angle's 2^-24, then one rounding to the type
        over = (got.double() - want).abs() - (EPS_HALF[dtype] * want.abs() + size * 2.0 ** -21)
        # below f16's normal range, 2^-14, half a step is 2^-25 and no longer 2^-11 of the
        # value: of 17 million results three there were off by up to 2.2e-8 more
        assert float(over.max()) <= (2.0 ** -25 if dtype == "f16" else 0)

    check(q[:tokens], first[:tokens, :heads])
    at = torch.from_numpy(table[seq, index // page].astype(np.int64)).cuda(), torch.from_numpy(index % page).cuda()
    check(kp[at[0], :, at[1]], first[:tokens, heads:heads + kv])
    assert torch.equal(vp[at[0], :, at[1]], first[:tokens, heads + kv:])
    for pool, old in zip((kp, vp), before):
        pool[at[0], :, at[1]] = old[at[0], :, at[1]]
        assert torch.equal(pool, old)


def timed(f, n=5):
    f()
    best = math.inf
    for _ in range(n):
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        f()
        b.record()
        torch.cuda.synchronize()
        best = min(best, a.elapsed_time(b))
    return best


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("q_len,kv_len", [((300,), (3000,)), ((1,) * 16, (4000,) * 16)])
@pytest.mark.parametrize("bad", [1, 40, 1000])
def test_rows_that_see_a_nan_cost_little(V, dtype, q_len, kv_len, bad):
    """They are NaN at once: only rows that do not see what is not finite beside
    their keys are worth doing again.  (Done again they took 20 to 260 times as long.)"""
    c = Case(V, torch, dtype, 8, 2, 128, 16, q_len, kv_len, seed=42, poison=False)
    want, clean = c.run(), timed(c.run)
    pages = torch.from_numpy(c.table[:, :bad // 16 + 1].astype(np.int64)).cuda()
    for s in range(c.n):
        c.vp[pages[s], :, :min(bad, 16), 7] = math.nan
    got = c.run()
    assert bool(torch.isnan(got[..., 7]).all())
    keep = [d for d in range(128) if d != 7]
    assert torch.equal(got[..., keep], want[..., keep])
    took = timed(c.run)
    assert took < 8 * clean
    c.kp[pages[0], 0, 0, 0] = math.nan  # and no scores
    assert bool(torch.isnan(c.run()[:q_len[0], :4]).all())
    assert timed(c.run) < 8 * clean


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("prefix", [0, 50])
@pytest.mark.parametrize("q_len,kv_len,window,sinks", [((90,), (400,), 0, 0), ((200, 3), (300, 60), 100, 4), ((1, 5), (300, 200), 64, 2)])
def test_many_values_that_are_not_finite(V, dtype, prefix, q_len, kv_len, window, sinks):
    """Values of 60 keys, of every kind, in and out of sight: each row has what its
    own keys add up to."""
    c = Case(V, torch, dtype, 8, 2, 64, 16, q_len, kv_len, window, sinks, prefix=prefix, seed=43, poison=False)
    rng = np.random.default_rng(44)
    for s in range(c.n):
        for i, j in enumerate(rng.permutation(kv_len[s])[:60]):
            c.v[s][j, i % 2, rng.integers(20)] = (math.nan, math.inf, -math.inf)[i % 3]
    for i in range(0, prefix, 9):
        c.pv[i, i % 2, rng.integers(20, 30)] = (math.inf, math.nan)[i % 2]
    live = c.table >= 0
    for s in range(c.n):
        for j in range(kv_len[s]):
            if live[s, j // 16]:
                c.vp[c.table[s, j // 16], :, j % 16] = c.v[s][j].cuda()
    for j in range(prefix):
        if c.pre[j // 16] >= 0:
            c.vp[c.pre[j // 16], :, j % 16] = c.pv[j].cuda()
    got = c.run().float().cpu().numpy()
    want, tol = c.expected()
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(np.isposinf(got), np.isposinf(want))
    ok = np.isfinite(want)
    assert np.array_equal(np.isneginf(got), np.isneginf(want)) and ok.any() and not ok.all()
    assert np.all(np.abs(got[ok] - want[ok]) <= tol[ok])


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("n", [1, 4, 70])
def test_keys_with_an_infinity(V, dtype, n):
    """A seen key whose score is -inf has no weight; the rows whose score with it is
    +inf are NaN."""
    c = Case(V, torch, dtype, 4, 1, 64, 16, (n,), (n + 300,), seed=45, poison=False)
    c.q_host[..., 5] = c.q_host[..., 5].abs() + 0.25
    c.q_host[-1, 1, 5] *= -1
    c.q = c.q_host.cuda()
    for j in (0, 77, 200):
        # as good as -inf to 64 bits too: a score of -300 and less
        c.k[0][j, 0, 5] = -10000.0
        c.kp[c.table[0, j // 16], 0, j % 16] = c.k[0][j, 0].cuda()
        c.kp[c.table[0, j // 16], 0, j % 16, 5] = -math.inf
    got = c.run()
    assert bool(torch.isnan(got[-1, 1]).all())
    got[-1, 1] = 0
    assert bool(torch.isfinite(got).all())
    want, tol = c.expected()
    want[-1, 1] = 0
    assert np.all(np.abs(got.double().cpu().numpy() - want) <= tol)


@pytest.mark.parametrize("step", [12.0, 25.0, 40.0, 70.0])
def test_scores_that_fall_again_and_again(V, step):
    """Every 64 keys far below the ones before, by up to 70 nats: the first, of value
    0, has all of the weight to 32 bits, and what follows adds up or is lost below the
    results' range, but nothing overflows."""
    c = dominated(V, "f16", 0.0, 0.0, (), heads=4, kv_heads=1, dim=128, q_len=(20,), kv_len=(1000,), seed=46)
    for i in range(0, 1000, 64):
        c.k[0][i:i + 64, :, 0] = max(300.0 - step * (i // 64), -300.0) * math.sqrt(c.dim) / 8.0
    c.v[0][:64] = 0.0
    store(c)
    check_dominated(c, c.run())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("q_len", [1, 90])
def test_the_stride_of_a_single_page_says_nothing(V, dtype, q_len):
    c = Case(V, torch, dtype, 8, 2, 64, 128, (q_len,), (100,), seed=47)
    only = int(c.table[0, 0])
    cache = V.PagedKvCache(c.kp[only:only + 1], c.vp[only:only + 1])
    batch = V.PagedBatch(c.q_start, c.kv, torch.zeros(1, 1, dtype=torch.int32, device="cuda"), c.tokens, q_len)
    for stride in (0, 8, 1 << 40):
        cache.desc.page_stride = stride
        c.check(V.paged_attention(cache, batch, c.q))
        batch.check()
