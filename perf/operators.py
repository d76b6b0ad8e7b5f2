"""What the paged-cache operators are measured on.

Three operators on one paged key/value cache: appending new keys and values
with the position rotation on the way (`append`), causal grouped-query
attention with a sliding window and sink tokens (`attn`), and the same for a
batch whose sequences share a prefix (`prefix`).

With `own` false, run() computes them in elementary torch operations; with
`own` true it calls the library's entry points.
"""
import importlib
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _case(name, op, dtype, heads, kv_heads, dim, page, seqs, q, kv, window=0, sinks=0, prefix=0, theta=1e6, base=0):
    """q and kv: (least, most) new tokens and cached tokens of a sequence, new ones included."""
    c = dict(op=op, dtype=dtype, heads=heads, kv_heads=kv_heads, dim=dim, page=page, seqs=seqs, q_lo=q[0], q_hi=q[1],
             kv_lo=kv[0], kv_hi=kv[1], window=window, sinks=sinks, prefix=prefix, theta=theta, base=base)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one stream's decode step: a single token's keys, values and queries; all latency
        _case("append_one_token", "append", "bf16", 32, 8, 128, 16, 1, (1, 1), (1537, 1537)),
        # a decode step of a large batch in the framework's own f32, far into long recordings
        _case("append_batch_f32", "append", "f32", 32, 8, 128, 64, 256, (1, 1), (1000, 8192), base=1000003),
        # ragged prompts filling their pages
        _case("append_prompts", "append", "bf16", 32, 8, 128, 16, 5, (911, 2600), (911, 2600)),
        # one stream's decode step at the benchmark's longer context
        _case("decode_one_stream", "attn", "bf16", 32, 8, 128, 16, 1, (1, 1), (1536, 1536), window=8192),
        # eight streams in f32, at the contexts of the multi-stream benchmark
        _case("decode_streams_f32", "attn", "f32", 32, 8, 128, 16, 8, (1, 1), (1036, 3513), window=8192),
        # a serving batch: short and very long sequences, the window with sinks, evicted pages gone
        _case("decode_serving", "attn", "f16", 32, 8, 128, 64, 96, (1, 1), (3, 32768), window=8192, sinks=4),
        # the benchmark's 512-id prompt in the framework's own f32
        _case("prompt_f32", "attn", "f32", 32, 8, 128, 16, 1, (512, 512), (512, 512), window=8192),
        # ragged whole prompts in one call
        _case("prefill_ragged", "attn", "bf16", 32, 8, 128, 32, 6, (300, 2500), (300, 2500)),
        # a chunk of a long prompt: the window and its sinks over 32 k cached tokens
        _case("chunk_long", "attn", "f16", 32, 8, 128, 64, 2, (2048, 2048), (24001, 32768), window=8192, sinks=16),
        # hypotheses of one recording that share its prompt; latency
        _case("prefix_nbest", "prefix", "bf16", 32, 8, 128, 16, 8, (1, 1), (1, 40), prefix=639),
        # a batch behind one long system prompt
        _case("prefix_batch", "prefix", "f16", 32, 8, 128, 32, 64, (1, 1), (1, 512), prefix=8192),
        # several drafted tokens a sequence, 32 k shared, the smaller head dimension
        _case("prefix_long", "prefix", "bf16", 64, 8, 64, 64, 128, (1, 4), (4, 256), prefix=32700),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        case = _drawn(rng)
        w = work(case)
        # f32 products run at a fraction of the 16-bit rate: no drawn case costs more than the largest listed ones
        if w["bytes"] <= 2.5e9 and w["flops"] <= (5e10 if case["dtype"] == "f32" else 5e11):
            return case


def _drawn(rng):
    op = rng.choice(["append", "attn_decode", "attn_prefill", "prefix"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 4, 4, 5, 7, 8])
    dim = rng.choice([64, 128, 128])
    page = rng.choice([8, 16, 32, 64, 128])
    theta = rng.choice([1e4, 1e6])
    if op == "append":
        seqs = _log(rng, 1, 256)
        q = _log(rng, 1, max(1, 8192 // seqs))
        kv = _log(rng, q, 16384)
        return _case("", "append", dtype, heads, kv_heads, dim, page, seqs, (1, q), (q, kv), theta=theta,
                     base=rng.choice([0, 0, _log(rng, 1, 4000000)]))
    if op == "attn_decode":
        seqs = _log(rng, 1, 96)
        kv = _log(rng, 5, min(32768, 1048576 // seqs))
        window = rng.choice([0, 8192, _log(rng, 1, 16384)])
        return _case("", "attn", dtype, heads, kv_heads, dim, page, seqs, (1, rng.choice([1, 1, 1, 5])), (5, kv),
                     window=window, sinks=rng.choice([0, 4, rng.randint(1, 200)]) if window else 0)
    if op == "attn_prefill":
        seqs = _log(rng, 1, 8)
        q = _log(rng, 16, (1024 if dtype == "f32" else 4096) // seqs)
        kv = _log(rng, q, 8192 if dtype == "f32" else 16384)
        window = rng.choice([0, 8192, _log(rng, 16, 8192)])
        return _case("", "attn", dtype, heads, kv_heads, dim, page, seqs, (max(1, q // 3), q), (q, kv),
                     window=window, sinks=rng.choice([0, 4, rng.randint(1, 200)]) if window else 0)
    seqs = _log(rng, 2, 128)
    q = rng.choice([1, 1, 1, 4])
    window = rng.choice([0, 0, _log(rng, 64, 16384)])
    return _case("", "prefix", dtype, heads, kv_heads, dim, page, seqs, (1, q), (q, _log(rng, q, 512)),
                 prefix=_log(rng, 20, 8192 if dtype == "f32" else 32768), window=window,
                 sinks=rng.choice([0, 4]) if window else 0)


def _spread(n, lo, hi, shift):
    """n lengths between lo and hi, spread and out of order; hi is among them."""
    got = [lo + int((hi - lo + 1) * ((0.6180339887498949 * i + shift) % 1.0)) for i in range(n)]
    got[n // 2] = hi
    return got


def _lengths(case):
    q = _spread(case["seqs"], case["q_lo"], case["q_hi"], 0.11)
    kv = _spread(case["seqs"], case["kv_lo"], case["kv_hi"], 0.83)
    return q, [max(a, b) for a, b in zip(q, kv)]


def _visible_keys(case, q_len, kv_len, prefix):
    """Keys of one sequence that some query sees, counted as (in the prefix, its own)."""
    first, last = prefix + kv_len - q_len, prefix + kv_len
    lo = max(0, first - case["window"] + 1) if case["window"] else 0
    sinks = min(case["sinks"], lo)
    shared = min(sinks, prefix) + max(0, prefix - lo)
    return shared, sinks + last - lo - shared


def _pairs(case, q_len, kv_len, prefix):
    """Visible (query, key) pairs of one sequence."""
    n = 0
    for i in range(q_len):
        p = prefix + kv_len - q_len + i
        lo = max(0, p - case["window"] + 1) if case["window"] else 0
        n += p + 1 - lo + min(case["sinks"], lo)
    return n


def work(case):
    q, kv = _lengths(case)
    size = 4 if case["dtype"] == "f32" else 2
    rows = sum(q) * case["dim"] * size
    if case["op"] == "append":
        elems = sum(q) * case["dim"] * (case["heads"] + 2 * case["kv_heads"])
        return {"bytes": 2 * elems * size, "flops": 3 * sum(q) * case["dim"] * (case["heads"] + case["kv_heads"])}
    keys = pairs = shared = 0
    for a, b in zip(q, kv):
        s, o = _visible_keys(case, a, b, case["prefix"])
        shared, keys = max(shared, s), keys + o
        pairs += _pairs(case, a, b, case["prefix"])
    return {"bytes": 2 * rows * case["heads"] + 2 * (keys + shared) * case["kv_heads"] * case["dim"] * size,
            "flops": 4 * case["dim"] * case["heads"] * pairs}


def _inputs(case, seed):
    """Host-side plan and device tensors of a case."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt, dim, page = DTYPES[case["dtype"]], case["dim"], case["page"]
    q_len, kv_len = _lengths(case)
    tokens = sum(q_len)
    prefix_pages = -(-case["prefix"] // page)
    width = max(-(-n // page) for n in kv_len)
    table = torch.full((case["seqs"], width), -1, dtype=torch.int64)
    used = prefix_pages
    for s, (a, b) in enumerate(zip(q_len, kv_len)):
        for j in range(-(-b // page)):
            # a page that lies between the sinks and every query's window has been given back
            gone = case["op"] == "attn" and case["window"] and j * page >= case["sinks"] and \
                (j + 1) * page <= b - a - case["window"] + 1
            if not gone:
                table[s, j] = used
                used += 1
    pages = used + 3
    order = torch.randperm(pages, generator=g, device="cuda").int()
    table = table.cuda()
    table = torch.where(table >= 0, order[table.clamp(min=0)], -1).int()
    starts = torch.tensor([0] + q_len).cumsum(0).int().cuda()
    # what a fused projection leaves: one row a token, queries, keys and values side by side
    qkv = torch.randn(tokens, (case["heads"] + 2 * case["kv_heads"]) * dim, generator=g, device="cuda")
    qkv[:, :case["heads"] * dim] *= 1.5
    qkv = qkv.to(dt)
    nq, nk = case["heads"] * dim, case["kv_heads"] * dim
    s = dict(case=case, q=qkv[:, :nq].unflatten(1, (-1, dim)), k_new=qkv[:, nq:nq + nk].unflatten(1, (-1, dim)),
             v_new=qkv[:, nq + nk:].unflatten(1, (-1, dim)), q_start=starts,
             kv_len=torch.tensor(kv_len, dtype=torch.int32).cuda(), table=table, tokens=tokens, max_q=max(q_len),
             max_kv=max(kv_len), q_len=q_len, kv_len_host=kv_len,
             k_pages=torch.randn(pages, case["kv_heads"], page, dim, generator=g, device="cuda", dtype=dt),
             v_pages=torch.randn(pages, case["kv_heads"], page, dim, generator=g, device="cuda", dtype=dt),
             first_pos=torch.full((case["seqs"],), case["base"], dtype=torch.int64, device="cuda"),
             prefix_pages=order[:prefix_pages].contiguous(),
             prefix_len=torch.tensor([case["prefix"]], dtype=torch.int32).cuda())
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        V = importlib.import_module("voxtral-rust_b200")
        # the handles that a program keeps: the layer's pool, and the batch that all layers share
        s["V"] = V
        s["cache"] = V.PagedKvCache(s["k_pages"], s["v_pages"])
        s["batch"] = V.PagedBatch(s["q_start"], s["kv_len"], s["table"], n_tokens=s["tokens"], max_q_len=s["max_q"],
                                  max_kv_len=s["max_kv"], first_pos=s["first_pos"])
    return s


def run(s):
    c = s["case"]
    if own:
        V = s["V"]
        if c["op"] == "append":
            q = V.paged_append_rope(s["cache"], s["batch"], s["k_new"], s["v_new"], c["theta"], q=s["q"])
            return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
        if c["op"] == "attn":
            return V.paged_attention(s["cache"], s["batch"], s["q"], sliding_window=c["window"], n_sinks=c["sinks"])
        return V.paged_prefix_attention(s["cache"], s["batch"], s["prefix_pages"], s["prefix_len"], c["prefix"], s["q"],
                                        sliding_window=c["window"], n_sinks=c["sinks"])
    if c["op"] == "append":
        return _plain_append(s)
    return _plain_attn(s) if c["op"] == "attn" else _plain_prefix(s)


# ---- plain forms ------------------------------------------------------------


def _token_rows(s):
    """Each token's sequence and its index in the sequence's cache."""
    t = torch.arange(s["tokens"], device="cuda")
    seq = torch.searchsorted(s["q_start"][1:], t.int(), right=True)
    index = s["kv_len"][seq].long() - s["q_start"][seq + 1].long() + t
    return t, seq, index


def _rotate(x, cos, sin):
    x = x.float()
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)


def _plain_append(s):
    c = s["case"]
    _, seq, index = _token_rows(s)
    pos = (s["first_pos"][seq] + index).double()
    freq = torch.pow(c["theta"], torch.arange(0, c["dim"], 2, device="cuda", dtype=torch.float64) * (-1.0 / c["dim"]))
    angle = (pos[:, None] * freq)[:, None, :]
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    page = s["table"][seq, index // c["page"]].long()
    slot = index % c["page"]
    s["k_pages"][page, :, slot] = _rotate(s["k_new"], cos, sin).to(s["k_pages"].dtype)
    s["v_pages"][page, :, slot] = s["v_new"]
    q = _rotate(s["q"], cos, sin).to(s["q"].dtype)
    return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _gather(pages, table):
    """Pages of each row of the table as [rows, heads, tokens, dim] in 32 bits."""
    got = pages[table.clamp(min=0).long()].transpose(1, 2)
    return got.flatten(2, 3).float()


def _seen(case, pos, key):
    seen = key <= pos
    if case["window"]:
        seen = seen & ((key < case["sinks"]) | (key > pos - case["window"]))
    return seen


def _own_scores(s, offset):
    """Scores of each sequence's padded queries against its own pages, masked: [seqs, kv_heads, group, queries, keys]."""
    c = s["case"]
    k = _gather(s["k_pages"], s["table"])
    i = torch.arange(s["max_q"], device="cuda")
    row = (s["q_start"][:-1, None].long() + i).clamp(max=s["tokens"] - 1)
    q = s["q"].float()[row].unflatten(2, (c["kv_heads"], -1)).permute(0, 2, 3, 1, 4)
    scores = torch.matmul(q.flatten(2, 3), k.transpose(-1, -2)).mul_(1.0 / math.sqrt(c["dim"]))
    q_len = (s["q_start"][1:] - s["q_start"][:-1]).long()
    pos = offset + (s["kv_len"].long() - q_len)[:, None] + i
    seen = _seen(c, pos[:, :, None], offset + torch.arange(k.shape[2], device="cuda"))
    return scores.unflatten(2, (-1, s["max_q"])).masked_fill_(~seen[:, None, None], -math.inf)


def _plain_attn(s):
    c = s["case"]
    scores = _own_scores(s, 0)
    top = scores.amax(-1, keepdim=True)
    p = scores.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.flatten(2, 3), _gather(s["v_pages"], s["table"])).unflatten(2, p.shape[2:4])
    out = out / torch.where(total == 0, 1.0, total)
    t, seq, _ = _token_rows(s)
    out = out.permute(0, 3, 1, 2, 4)[seq, t - s["q_start"][seq]]
    return out.flatten(1, 2).to(DTYPES[c["dtype"]])


def _plain_prefix(s):
    c = s["case"]
    t, seq, index = _token_rows(s)
    offset = c["prefix"]
    k = _gather(s["k_pages"], s["prefix_pages"][None])[0, :, :offset]
    v = _gather(s["v_pages"], s["prefix_pages"][None])[0, :, :offset]
    q = s["q"].float().unflatten(1, (c["kv_heads"], -1)).permute(1, 2, 0, 3)
    shared = torch.matmul(q.flatten(1, 2), k.transpose(-1, -2)).mul_(1.0 / math.sqrt(c["dim"]))
    seen = _seen(c, (offset + index)[:, None], torch.arange(offset, device="cuda"))
    shared = shared.unflatten(1, (-1, s["tokens"])).masked_fill_(~seen, -math.inf)
    mine = _own_scores(s, offset)
    top = torch.maximum(shared.amax(-1), mine.permute(0, 3, 1, 2, 4)[seq, t - s["q_start"][seq]].amax(-1).permute(1, 2, 0))
    top = torch.where(top == -math.inf, 0.0, top)
    shared = shared.sub_(top[..., None]).exp_()
    i = torch.arange(s["max_q"], device="cuda")
    row = (s["q_start"][:-1, None].long() + i).clamp(max=s["tokens"] - 1)
    mine = mine.sub_(top.permute(2, 0, 1)[row].permute(0, 2, 3, 1)[..., None]).exp_()
    own_out = torch.matmul(mine.flatten(2, 3), _gather(s["v_pages"], s["table"])).unflatten(2, mine.shape[2:4])
    place = t - s["q_start"][seq]
    out = torch.matmul(shared.flatten(1, 2), v).unflatten(1, (-1, s["tokens"])).permute(2, 0, 1, 3)
    out = out + own_out.permute(0, 3, 1, 2, 4)[seq, place]
    total = shared.sum(-1).permute(2, 0, 1) + mine.sum(-1).permute(0, 3, 1, 2)[seq, place]
    out = out / torch.where(total == 0, 1.0, total)[..., None]
    return out.flatten(1, 2).to(DTYPES[c["dtype"]])


# ---- the definition in 64 bits ----------------------------------------------


def exact(case, seed):
    global own
    kept, own = own, False
    try:
        s = _inputs(case, seed)
    finally:
        own = kept
    if case["op"] == "append":
        half = case["dim"] // 2
        freq = torch.exp(torch.arange(half, dtype=torch.float64) * (-2.0 * math.log(case["theta"]) / case["dim"])).cuda()
        k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
        rotated = {}
        positions = [case["base"] + b - a + i for a, b in zip(s["q_len"], s["kv_len_host"]) for i in range(a)]
        turn = torch.tensor(positions, dtype=torch.float64).cuda()[:, None] * freq
        turn = torch.polar(torch.ones_like(turn), turn)[:, None, :]
        for name in ("q", "k_new"):
            z = torch.view_as_complex(s[name].double().unflatten(-1, (half, 2)).contiguous())
            rotated[name] = torch.view_as_real(z * turn).flatten(-2)
        at = 0
        for n, (a, b) in enumerate(zip(s["q_len"], s["kv_len_host"])):
            where = torch.arange(b - a, b).cuda()
            page = s["table"][n].long()[where // case["page"]]
            k_pages[page, :, where % case["page"]] = rotated["k_new"][at:at + a]
            v_pages[page, :, where % case["page"]] = s["v_new"][at:at + a].double()
            at += a
        return {"q": rotated["q"], "k_pages": k_pages, "v_pages": v_pages}
    out = torch.zeros(s["tokens"], case["heads"], case["dim"], dtype=torch.float64, device="cuda")
    group, at = case["heads"] // case["kv_heads"], 0
    shared = s["prefix_pages"].long()
    for n, (a, b) in enumerate(zip(s["q_len"], s["kv_len_host"])):
        mine = s["table"][n, :-(-b // case["page"])].long().clamp(min=0)
        pos = case["prefix"] + torch.arange(b - a, b, device="cuda")
        for h in range(case["kv_heads"]):
            keys, values = (torch.cat((x[shared, h].flatten(0, 1)[:case["prefix"]], x[mine, h].flatten(0, 1)[:b])).double()
                            for x in (s["k_pages"], s["v_pages"]))
            j = torch.arange(keys.shape[0], device="cuda")
            hidden = j[None] > pos[:, None]
            if case["window"]:
                hidden |= (j[None] <= pos[:, None] - case["window"]) & (j[None] >= case["sinks"])
            q = s["q"][at:at + a, h * group:(h + 1) * group].double()
            w = torch.einsum("tgd,jd->gtj", q, keys) / case["dim"] ** 0.5
            w = torch.softmax(w.masked_fill(hidden, -math.inf), -1)
            out[at:at + a, h * group:(h + 1) * group] = torch.einsum("gtj,jd->tgd", w, values)
        at += a
    return out
