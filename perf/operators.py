"""The operators over paged rows -- a paged cache and its page operations, attention of one new token over it, latent attention in its absorbed
and its expanded form -- as they are measured: the cases, their inputs, the plain form of each operator (elementary torch operations in float32)
and its definition in 64 bits.

`own` says which side `run` computes: False = the plain form, True = the calls of scalablevectorsearch_amd."""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one user's next token behind a short prompt: latency decides
        dict(name="attend_one", op="attend", dtype="bf16", batch=1, heads=32, kv_heads=8, dim=128, value_dim=128, page=16, length=777, ragged=False, holes=0.0),
        # a serving batch of ragged conversations, grouped heads
        dict(name="attend_batch", op="attend", dtype="f16", batch=64, heads=32, kv_heads=8, dim=128, value_dim=128, page=16, length=8191, ragged=True, holes=0.0),
        # few long documents: the work is split over the cache's length
        dict(name="attend_long", op="attend", dtype="bf16", batch=4, heads=64, kv_heads=8, dim=128, value_dim=128, page=64, length=131071, ragged=False, holes=0.0),
        # attention over the 100 rows that a search returned (pages of one row, float32 rows of 96 components, some answers short of 100)
        dict(name="attend_neighbours", op="attend", dtype="f32", batch=2048, heads=1, kv_heads=1, dim=96, value_dim=96, page=1, length=100, ragged=False, holes=0.02),
        # latent attention, absorbed form: one conversation on a model of 16 heads
        dict(name="latent_one", op="latent", dtype="bf16", batch=1, heads=16, dim=576, value_dim=512, page=16, length=4097, ragged=False, holes=0.0),
        # the same for a serving batch on a model of 128 heads
        dict(name="latent_batch", op="latent", dtype="bf16", batch=32, heads=128, dim=576, value_dim=512, page=64, length=8192, ragged=True, holes=0.0),
        # latent attention, expanded form: three short prompts in one batch
        dict(name="prompt_small", op="prompt", dtype="f16", sequences=3, tokens=333, rows=333, heads=16, nope=128, rope=64, value_dim=128, rank=512),
        # one long prompt whose second half is new
        dict(name="prompt_long", op="prompt", dtype="bf16", sequences=1, tokens=4095, rows=8190, heads=32, nope=128, rope=64, value_dim=128, rank=512),
        # one layer's rows of a decoding step, into slots that were taken before
        dict(name="write_step", op="write", dtype="bf16", layers=1, sequences=128, tokens=128, heads=8, dim=128, value_dim=128, page=16),
        # prompts taken into the cache: their pages are taken, then each layer's rows are written
        dict(name="write_prompt", op="fill", dtype="f32", layers=2, sequences=8, tokens=16381, heads=8, dim=128, value_dim=128, page=16),
        # eight samples of each prompt: the prompt's full pages are shared, the last one is copied, each sample gets its first token
        dict(name="fork_step", op="fork", dtype="bf16", layers=4, sequences=8, children=8, length=1023, heads=8, dim=128, value_dim=128, page=16),
        # sequences copied whole, some of them freed, the holes closed
        dict(name="copy_compact", op="compact", dtype="f16", layers=2, sequences=16, length=1019, heads=8, dim=128, value_dim=128, page=16),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "neighbours", "latent", "latent", "prompt", "prompt", "write", "fill", "fork", "compact"])
    dtype = rng.choice(["f32", "f16", "bf16", "f16", "bf16"])
    if op == "attend":
        kv = rng.choice([1, 2, 4, 8])
        dim = rng.choice([64, 80, 96, 128, 128, 192, 256])
        batch, page = _log(rng, 1, 128), rng.choice([8, 16, 32, 64, 128])
        length = _log(rng, 1, max(16, min(100000, (1 << 29) // (batch * kv * dim))))
        return dict(op="attend", dtype=dtype, batch=batch, heads=kv * rng.choice([1, 2, 3, 4, 7, 8, 16]), kv_heads=kv, dim=dim, value_dim=dim, page=page,
                    length=length, ragged=rng.random() < 0.7, holes=0.0)
    if op == "neighbours":
        return dict(op="attend", dtype=dtype, batch=_log(rng, 1, 4000), heads=rng.choice([1, 1, 4]), kv_heads=1, dim=rng.choice([96, 100, 128, 200]),
                    value_dim=0, page=1, length=_log(rng, 10, 200), ragged=False, holes=rng.choice([0.0, 0.05, 0.5]))
    if op == "latent":
        batch = _log(rng, 1, 64)
        rank = rng.choice([256, 512, 512])
        return dict(op="latent", dtype=rng.choice(["f16", "bf16", "bf16", "f32"]), batch=batch, heads=rng.choice([8, 16, 20, 32, 64, 128]), dim=rank + rng.choice([32, 64, 64]),
                    value_dim=rank, page=rng.choice([1, 16, 32, 64]), length=_log(rng, 1, min(60000, 200000 // batch)), ragged=rng.random() < 0.7, holes=0.0)
    if op == "prompt":
        sequences, heads = rng.choice([1, 1, 2, 3, 7]), rng.choice([8, 16, 16, 32])
        tokens = _log(rng, 8, 2048)
        return dict(op="prompt", dtype=dtype, sequences=sequences, tokens=max(tokens, sequences), rows=max(tokens, sequences) + rng.choice([0, 0, _log(rng, 1, 2000)]),
                    heads=heads, nope=rng.choice([64, 128]), rope=rng.choice([32, 64]), value_dim=rng.choice([64, 128]), rank=rng.choice([256, 512]))
    heads, dim, page = rng.choice([1, 2, 8]), rng.choice([64, 96, 128, 256]), rng.choice([8, 16, 32, 64])
    if op == "write":
        sequences = _log(rng, 1, 512)
        return dict(op="write", dtype=dtype, layers=1, sequences=sequences, tokens=sequences, heads=heads, dim=dim, value_dim=dim, page=page)
    if op == "fill":
        sequences = rng.choice([1, 2, 5, 16])
        return dict(op="fill", dtype=dtype, layers=rng.choice([1, 2, 4]), sequences=sequences, tokens=_log(rng, sequences, 12000), heads=heads, dim=dim, value_dim=dim, page=page)
    if op == "fork":
        return dict(op="fork", dtype=dtype, layers=rng.choice([1, 2, 4]), sequences=_log(rng, 1, 32), children=rng.choice([1, 2, 4, 8]), length=_log(rng, 1, 4000),
                    heads=heads, dim=dim, value_dim=dim, page=page)
    return dict(op="compact", dtype=dtype, layers=rng.choice([1, 2]), sequences=_log(rng, 1, 24), length=_log(rng, 1, 1200), heads=heads, dim=dim, value_dim=dim, page=page)


def _value_dim(case):
    return case["value_dim"] or case["dim"]


def _lengths(case, g):
    """The sequences' lengths, on the host: all alike, or spread evenly from one token to the longest."""
    n, longest = case["batch"], case["length"]
    if not case["ragged"]:
        return torch.full((n,), longest, dtype=torch.int32)
    got = torch.randint(1, longest + 1, (n,), generator=g, dtype=torch.int32)
    got[0] = longest
    return got


def _split(total, n, g):
    """n counts of at least one with the given sum, as offsets."""
    cuts = (torch.randperm(total - 1, generator=g)[: n - 1] + 1).sort().values if n > 1 else torch.zeros(0, dtype=torch.int64)
    return torch.cat([torch.zeros(1, dtype=torch.int64), cuts, torch.tensor([total])]).to(torch.int32)


def prepare(case, seed):
    g = torch.Generator().manual_seed(seed)
    gg = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=gg, device="cuda", dtype=torch.float32).to(dtype) if math.prod(shape) < 1 << 28 else torch.randn(shape, generator=gg, device="cuda", dtype=dtype)

    st = {"case": case}
    if case["op"] in ("attend", "latent"):
        lengths = _lengths(case, g)
        page, n = case["page"], case["batch"]
        columns = -(-int(lengths.max()) // page)
        if page == 1 and case["op"] == "attend":  # rows of an index; which of them a query attends to came out of a search
            pages = 20000
            table = torch.randint(0, pages, (n, columns), generator=g, dtype=torch.int32)
            table[torch.rand((n, columns), generator=g) < case["holes"]] = -1
        else:
            taken = -(-lengths.long() // page)
            pages = int(taken.sum()) + 7
            table = torch.full((n, columns), -1, dtype=torch.int32)
            table[torch.arange(columns)[None] < taken[:, None]] = torch.randperm(pages, generator=g)[: int(taken.sum())].to(torch.int32)
        st |= {"queries": normal(n, case["heads"], case["dim"]), "keys": normal(pages, case.get("kv_heads", 1), page, case["dim"]), "table": table.cuda(), "lengths": lengths.cuda()}
        # the first columns of a latent row are its value; a neighbour's row is key and value at once
        st["values"] = normal(pages, case["kv_heads"], page, case["value_dim"]) if case["op"] == "attend" and case["value_dim"] else None
        if case["op"] == "latent":  # queries in the latent space are a head's query times its up-projection
            st["queries"] *= 0.8
        return st
    if case["op"] == "prompt":
        h, rank = case["heads"], case["rank"]
        n = case["sequences"]
        q = _split(case["tokens"], n, g)
        old = case["rows"] - case["tokens"]
        r = q + (torch.arange(n + 1) * old // n).to(torch.int32)  # rows that were there before the prompt's own
        return st | {"queries": normal(case["tokens"], h, case["nope"] + case["rope"]), "rows": normal(case["rows"], rank + case["rope"]),
                     "w_key": normal(h, case["nope"], rank) * rank**-0.5, "w_value": normal(h, case["value_dim"], rank) * rank**-0.5, "query_offsets": q.cuda(), "row_offsets": r.cuda()}
    # a cache that holds some sequences already, its pages in no order
    page, n, layers = case["page"], case["sequences"], case["layers"]
    if case["op"] in ("write", "fill"):
        live, more = 0, case["tokens"] // page + 2 * n
        seqs, offsets = torch.arange(n, dtype=torch.int32), _split(case["tokens"], n, g)
        slots_of, longest = n, case["tokens"]
    elif case["op"] == "fork":
        live, more = n, n * case["children"] * 2
        slots_of, longest = n * (1 + case["children"]), case["length"] + 1
    else:
        live, more = 2 * n, 2 * n * -(-case["length"] // page) + 3  # a copy of each
        slots_of, longest = 4 * n, case["length"]
    columns = -(-longest // page)
    lengths = torch.zeros(slots_of, dtype=torch.int32)
    if live:
        lengths[:live] = torch.randint(max(1, longest * 3 // 4), longest, (live,), generator=g, dtype=torch.int32) if longest > 1 else 1
    taken = -(-lengths.long() // page)
    used, pages = int(taken.sum()), live * columns + more
    # a fragmented pool, but for `compact`, which leaves a dense one behind at the end of every pass
    order = torch.randperm(used if case["op"] == "compact" else pages, generator=g)[:used].to(torch.int32)
    table = torch.full((slots_of, columns), -1, dtype=torch.int32)
    table[torch.arange(columns)[None] < taken[:, None]] = order
    refs = torch.zeros(pages, dtype=torch.int32)
    refs[order.long()] = 1
    st |= {"keys": normal(layers, pages, case["heads"], page, case["dim"]), "values": normal(layers, pages, case["heads"], page, case["value_dim"]), "table": table.cuda(),
           "lengths": lengths.cuda(), "refs": refs.cuda()}
    if case["op"] in ("write", "fill"):
        st |= {"seqs": seqs.cuda(), "offsets": offsets.cuda(), "n_tokens": case["tokens"]}
    elif case["op"] == "fork":
        children = n * case["children"]
        st |= {"sources": torch.arange(n, dtype=torch.int32).repeat_interleave(case["children"]).cuda(), "targets": torch.arange(n, n + children, dtype=torch.int32).cuda(),
               "offsets": torch.arange(children + 1, dtype=torch.int32).cuda(), "n_tokens": children}
    else:
        a = torch.arange(n, dtype=torch.int32).cuda()
        st |= {"a": a, "b": a + n, "x": a + 2 * n, "y": a + 3 * n}
    if "n_tokens" in st:
        st |= {"new_keys": normal(layers, st["n_tokens"], case["heads"], case["dim"]), "new_values": normal(layers, st["n_tokens"], case["heads"], case["value_dim"])}
    if case["op"] == "write":  # slots that the step's bookkeeping gave out, once for all layers
        st["slots"] = torch.randperm(pages * page, generator=g)[: case["tokens"]].cuda()
    if own:  # the handle on the cache that a program keeps
        import scalablevectorsearch_amd as svs

        st["cache"] = svs.PagedCache.from_device(st["keys"], st["values"], st["table"], st["lengths"], st["refs"])
    return st


def run(st):
    case = st["case"]
    op = case["op"]
    if own:
        import scalablevectorsearch_amd as svs

        if op == "attend":
            out, lse = svs.paged_attention(st["queries"], st["keys"], st["values"], st["table"], st["lengths"], value_dim=_value_dim(case), return_lse=True)
            return {"out": out, "lse": lse}
        if op == "latent":
            out, lse = svs.latent_attention(st["queries"], st["keys"], st["table"], st["lengths"], value_dim=case["value_dim"], return_lse=True)
            return {"out": out, "lse": lse}
        if op == "prompt":
            return {"out": svs.latent_attention_expanded(st["queries"], st["rows"], st["w_key"], st["w_value"], st["query_offsets"], st["row_offsets"])}
        cache = st["cache"]
        free, extend, write, copy, fork, compact = cache.free, cache.extend, cache.write, cache.copy, cache.fork, cache.compact
    else:
        if op in ("attend", "latent"):
            return _attend_plain(st, _value_dim(case))
        if op == "prompt":
            return _prompt_plain(st, case)
        free, extend, write = (lambda *a: _free(st, *a)), (lambda *a: _extend(st, *a)), (lambda *a, **k: _write(st, *a, **k))
        copy, fork, compact = (lambda *a: _copy(st, *a, share=False)), (lambda *a: _copy(st, *a, share=True)), (lambda: _compact(st))
    if op == "write":
        write(st["slots"], st["new_keys"][0], st["new_values"][0])
        return {"keys": st["keys"], "values": st["values"]}
    got = {}
    if op == "fill":
        free(st["seqs"])
        got["slots"] = extend(st["seqs"], st["offsets"], st["n_tokens"])
    elif op == "fork":
        free(st["targets"])
        fork(st["sources"], st["targets"])
        got["slots"] = extend(st["targets"], st["offsets"], st["n_tokens"])
    else:
        free(st["y"])
        copy(st["a"], st["x"])
        copy(st["b"], st["y"])
        free(st["x"])
        got["moved"] = compact()
    for layer in range(case["layers"] if "slots" in got else 0):
        write(got["slots"], st["new_keys"][layer], st["new_values"][layer], layer=layer)
    return got | {k: st[k] for k in ("keys", "values", "table", "lengths", "refs")}


# ---- plain forms ------------------------------------------------------------------------------------------------------------------------------


def _attend_plain(st, value_dim):
    q, keys, values, table = st["queries"], st["keys"], st["values"], st["table"]
    n, heads, dim = q.shape
    pages, kv, page, _ = keys.shape
    there = (table >= 0) & (table < pages)
    at = torch.where(there, table, 0).long()
    length = table.shape[1] * page

    def rows(x):
        return x[at].float().permute(0, 2, 1, 3, 4).reshape(n, kv, length, x.shape[-1])

    k = rows(keys)
    v = rows(values) if values is not None else k[..., :value_dim]
    live = (torch.arange(length, device=q.device)[None] < st["lengths"][:, None]) & there.repeat_interleave(page, 1)
    s = torch.matmul(q.float().view(n, kv, heads // kv, dim), k.transpose(-1, -2)) * dim**-0.5
    s = s.masked_fill(~live[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v.masked_fill(~live[:, None, :, None], 0.0)) / torch.where(total > 0, total, 1.0)
    return {"out": out.reshape(n, heads, value_dim).to(q.dtype), "lse": (top + torch.log(total)).reshape(n, heads)}


def _prompt_plain(st, case):
    q, rows, rank, nope = st["queries"].float(), st["rows"].float(), case["rank"], case["nope"]
    qo, ro = st["query_offsets"].long(), st["row_offsets"].long()
    heads = case["heads"]
    k = torch.matmul(rows[:, :rank], st["w_key"].float().transpose(1, 2))  # heads, rows, nope
    v = torch.matmul(rows[:, :rank], st["w_value"].float().transpose(1, 2))
    k = torch.cat([k, rows[None, :, rank:].expand(heads, -1, -1)], -1)
    s = torch.matmul(q.permute(1, 0, 2), k.transpose(1, 2)) * (q.shape[-1] ** -0.5)
    t, r = torch.arange(q.shape[0], device=q.device), torch.arange(rows.shape[0], device=q.device)
    of_t, of_r = torch.bucketize(t, qo[1:], right=True), torch.bucketize(r, ro[1:], right=True)
    last = ro[of_t + 1] - qo[of_t + 1] + t  # the last row that a token sees: its own
    s = s.masked_fill(~((of_t[:, None] == of_r[None]) & (r[None] <= last[:, None])), -math.inf)
    s -= s.amax(-1, keepdim=True)
    p = s.exp_()
    out = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    return {"out": out.permute(1, 0, 2).to(st["queries"].dtype)}


def _take(st, need):
    """The lowest free pages, as many as are needed: (each entry's first rank, the pages by rank)."""
    first = need.cumsum(0) - need
    return first, (st["refs"] == 0).nonzero()[:, 0]


def _free(st, seqs):
    seqs = seqs.long()
    gone = st["table"][seqs]
    gone = gone[gone >= 0].long()
    st["refs"].index_add_(0, gone, torch.full_like(gone, -1, dtype=torch.int32))
    st["table"][seqs] = -1
    st["lengths"][seqs] = 0


def _extend(st, seqs, offsets, n_tokens):
    seqs, offsets, page = seqs.long(), offsets.long(), st["keys"].shape[3]
    old, count = st["lengths"][seqs].long(), offsets[1:] - offsets[:-1]
    have = (old + page - 1) // page
    need = (old + count + page - 1) // page - have
    first, pages = _take(st, need)
    entry = torch.arange(len(seqs), device=seqs.device).repeat_interleave(need)
    rank = torch.arange(len(entry), device=seqs.device)
    pages = pages[: len(entry)]
    st["table"][seqs[entry], have[entry] + rank - first[entry]] = pages.to(torch.int32)
    st["refs"][pages] = 1
    st["lengths"][seqs] = (old + count).to(torch.int32)
    entry = torch.arange(len(seqs), device=seqs.device).repeat_interleave(count)
    at = old[entry] + torch.arange(n_tokens, device=seqs.device) - offsets[entry]
    return st["table"][seqs[entry], at // page].long() * page + at % page


def _write(st, slots, keys, values, layer=0):
    page = st["keys"].shape[3]
    st["keys"][layer, slots // page, :, slots % page] = keys
    st["values"][layer, slots // page, :, slots % page] = values


def _copy(st, sources, targets, share):
    sources, targets, page = sources.long(), targets.long(), st["keys"].shape[3]
    length = st["lengths"][sources].long()
    whole = length // page
    start = whole if share else torch.zeros_like(whole)
    need = (length + page - 1) // page - start
    first, pages = _take(st, need)
    entry = torch.arange(len(sources), device=sources.device).repeat_interleave(need)
    column = start[entry] + torch.arange(len(entry), device=sources.device) - first[entry]
    pages = pages[: len(entry)]
    old = st["table"][sources[entry], column].long()
    shared = st["table"][sources]
    shared = shared.masked_fill(torch.arange(shared.shape[1], device=sources.device)[None] >= start[:, None], -1)
    st["table"][targets] = shared
    st["table"][targets[entry], column] = pages.to(torch.int32)
    shared = shared[shared >= 0].long()
    st["refs"].index_add_(0, shared, torch.ones_like(shared, dtype=torch.int32))
    st["refs"][pages] = 1
    st["lengths"][targets] = length.to(torch.int32)
    live = (torch.arange(page, device=sources.device)[None] < (length[entry] - column * page)[:, None])[None, :, None, :, None]
    for x in (st["keys"], st["values"]):
        x[:, pages] = torch.where(live, x[:, old], x[:, pages])


def _compact(st):
    used = st["refs"] > 0
    count = int(used.sum())
    to, old = (~used[:count]).nonzero()[:, 0], used[count:].nonzero()[:, 0] + count
    moved = torch.where(used, torch.arange(len(used), device=used.device), -1).to(torch.int32)
    moved[old] = to.to(torch.int32)
    for x in (st["keys"], st["values"]):
        x[:, to] = x[:, old]
    st["refs"][to] = st["refs"][old]
    st["refs"][old] = 0
    st["table"][:] = torch.where(st["table"] >= 0, moved[st["table"].clamp(min=0).long()], -1)
    return moved


# ---- definitions in 64 bits -------------------------------------------------------------------------------------------------------------------


def exact(case, seed):
    """softmax(scale * q . k over the rows that are there) times their values, sequence by sequence and head by head. Page operations compute
    whole numbers and move rows: they have no value here."""
    global own
    if case["op"] not in ("attend", "latent", "prompt"):
        return None
    was, own = own, False
    st = prepare(case, seed)
    own = was
    q = st["queries"].double()
    if case["op"] == "prompt":
        rank = case["rank"]
        out = torch.zeros(q.shape[0], case["heads"], case["value_dim"], dtype=torch.float64, device="cuda")
        qo, ro = st["query_offsets"].tolist(), st["row_offsets"].tolist()
        for i in range(case["sequences"]):
            c = st["rows"][ro[i]:ro[i + 1]].double()
            nq, nr = qo[i + 1] - qo[i], ro[i + 1] - ro[i]
            seen = torch.ones(nq, nr, dtype=torch.bool, device="cuda").tril(nr - nq)
            for h in range(case["heads"]):
                qh = q[qo[i]:qo[i + 1], h]
                s = (qh[:, : case["nope"]] @ st["w_key"][h].double()) @ c[:, :rank].T + qh[:, case["nope"]:] @ c[:, rank:].T  # w_key applied to the query, not to the rows
                p = torch.softmax((s / math.sqrt(q.shape[-1])).masked_fill(~seen, -math.inf), -1)
                out[qo[i]:qo[i + 1], h] = (p @ c[:, :rank]) @ st["w_value"][h].double().T
        return {"out": out}
    n, heads, dim = q.shape
    dv = _value_dim(case)
    kv, page = st["keys"].shape[1], st["keys"].shape[2]
    out = torch.zeros(n, heads, dv, dtype=torch.float64, device="cuda")
    lse = torch.full((n, heads), -math.inf, dtype=torch.float64, device="cuda")
    if page == 1 and n > 200:  # many short lists of rows: all at once
        table = st["table"].long()
        k = st["keys"][table.clamp(min=0), :, 0].double()  # n, rows, kv, dim
        v = st["values"][table.clamp(min=0), :, 0].double() if st["values"] is not None else k[..., :dv]
        k, v = (x.repeat_interleave(heads // kv, 2) for x in (k, v))
        s = (q[:, None] * k).sum(-1) / math.sqrt(dim)
        s[table < 0] = -math.inf
        lse = torch.logsumexp(s, 1)
        return {"out": (torch.exp(s - lse[:, None])[..., None] * v).sum(1).nan_to_num(0.0), "lse": lse}
    for b, length in enumerate(st["lengths"].tolist()):
        at = torch.arange(length, device="cuda")
        of = st["table"][b].long()[at // page]
        at, of = at[of >= 0], of[of >= 0]
        if not len(at):
            continue
        for h in range(kv):
            k = st["keys"][of, h, at % page].double()
            v = st["values"][of, h, at % page].double() if st["values"] is not None else k[:, :dv]
            mine = slice(h * (heads // kv), (h + 1) * (heads // kv))
            s = q[b, mine] @ k.T / math.sqrt(dim)
            lse[b, mine] = torch.logsumexp(s, -1)
            out[b, mine] = torch.softmax(s, -1) @ v
    return {"out": out, "lse": lse}


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] in ("attend", "latent"):
        n, dv, kv = case["batch"], _value_dim(case), case.get("kv_heads", 1)
        tokens = n * case["length"] * (0.5 if case["ragged"] else 1.0) * (1 - case["holes"])
        stored = case["dim"] + (dv if case["op"] == "attend" and case["value_dim"] else 0)
        rows = min(tokens, 20000) if case["page"] == 1 and case["op"] == "attend" else tokens  # neighbours' rows are shared between queries
        return {"bytes": rows * kv * stored * size + n * case["heads"] * ((case["dim"] + dv) * size + 4) + 4 * n * (case["length"] / case["page"]),
                "flops": 2.0 * tokens * case["heads"] * (case["dim"] + dv)}
    if case["op"] == "prompt":
        n, h, t, r, k, v = case["sequences"], case["heads"], case["tokens"], case["rows"], case["nope"] + case["rope"], case["value_dim"]
        pairs = (t / n) * (r / n - t / n / 2) * n
        return {"bytes": size * (t * h * (k + v) + r * (case["rank"] + case["rope"]) + h * (case["nope"] + v) * case["rank"]),
                "flops": 2.0 * h * (pairs * (k + v) + r * case["rank"] * (case["nope"] + v))}
    row = case["layers"] * case["heads"] * (case["dim"] + case["value_dim"]) * size
    if case["op"] in ("write", "fill"):
        return {"bytes": 2 * case["tokens"] * row + 8 * case["tokens"], "flops": 0}
    n, length = case["sequences"], case["length"] * 7 / 8
    if case["op"] == "fork":
        return {"bytes": n * case["children"] * (2 * (case["page"] / 2 + 1) * row + 4 * 4 * length / case["page"]), "flops": 0}
    return {"bytes": 3 * 2 * n * length * row, "flops": 0}
