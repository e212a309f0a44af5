"""Cases and plain forms of the prompt and cache operators of this framework, for timing and for checking.

Three operators around the paged cache ``[pages, P, Hkv, D]``:

* ``prefill`` -- causal or full attention of packed queries over packed keys or over the paged cache
  (``gqa_fwd_batch_prefill``);
* ``shared``  -- one decode step of sequences that share long prefixes (``gqa_fwd_batch_decode_shared_prefix``);
* ``pages``   -- copying, forking + freeing and compacting the pages of a cache (``paged_kv_copy``, ``paged_kv_fork``,
  ``paged_kv_free``, ``paged_kv_compact``).

``run`` computes an operator from elementary torch operations in 32 bits, or, where ``own`` is true, makes the calls that a
user of the framework makes.  ``exact`` computes the attention results from the definition in 64 bits.
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
ROWS_AT_ONCE = 1024        # query rows per slab of scores in the plain form


# ------------------------------------------------------------------------------------------------ cases

def _ints(text):
    """"5 7x3" -> [5, 7, 7, 7]: lengths are given as text."""
    out = []
    for word in str(text).split():
        n, _, times = word.partition("x")
        out += [int(n)] * (int(times) if times else 1)
    return out


def _prefill(name, q_lens, kv_lens, heads, kv_heads, dim, dtype, page=0, fp8=False, causal=True, soft_cap=0.0):
    return {"name": name, "kind": "prefill", "q_lens": q_lens, "kv_lens": kv_lens, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "dtype": dtype, "page": page, "fp8": fp8, "causal": causal, "soft_cap": soft_cap}


def _shared(name, prefix_lens, members, kv_lens, heads, kv_heads, dim, dtype, page, fp8=False, soft_cap=0.0):
    return {"name": name, "kind": "shared", "prefix_lens": prefix_lens, "members": members, "kv_lens": kv_lens,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "page": page, "fp8": fp8,
            "soft_cap": soft_cap}


def _pages(name, action, layers, pages, page, kv_heads, dim, dtype, rows, length, count):
    return {"name": name, "kind": "pages", "action": action, "layers": layers, "pages": pages, "page": page,
            "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "rows": rows, "length": length, "count": count}


def listed():
    return [
        # one short prompt of an interactive request: a single launch, latency is all that counts
        _prefill("prefill_one_short", "77", "77", 8, 2, 128, "fp16"),
        # a batch of prompts of different lengths, packed one behind the other, odd lengths among them
        _prefill("prefill_ragged", "33 1999 512 1 1024 777 2048 130 64 1500 350 95", "33 1999 512 1 1024 777 2048 130 64 "
                 "1500 350 95", 32, 8, 128, "bf16"),
        # one long document: the matrix products dominate everything else
        _prefill("prefill_long", "16384", "16384", 32, 8, 128, "bf16"),
        # chunks of long prompts against what an fp8 cache holds of them already
        _prefill("prefill_chunks_fp8", "512x3 401", "16384 9000 4608 12345", 64, 8, 128, "bf16", page=16, fp8=True),
        # drafted tokens of a speculative decoder checked in one pass: few rows, long caches, bound by memory
        _prefill("prefill_drafts", "5x8", "8192 8197 8001 7777 8192 6500 8100 8000", 32, 8, 128, "bf16", page=16),
        # a handful of requests behind one system prompt: the smallest step
        _shared("shared_few", "1000", "5", "17 60 1 33 48", 32, 8, 128, "bf16", 16),
        # a serving batch behind one long prompt (a document that many questions are asked about)
        _shared("shared_batch", "8192", "64", "64 1024 300 511 16 800 129 640 " * 8, 32, 8, 128, "bf16", 16),
        # four groups of different sizes on an fp8 cache, each with its own long prefix
        _shared("shared_groups_fp8", "16384 12000 8193 4096", "48 40 8 32", "256 1000 77 2048 512 129 1600 33 " * 16, 64, 8,
                128, "bf16", 16, fp8=True),
        # pages of one cache swapped for others in every layer (prefix reuse, defragmentation by the caller)
        _pages("pages_copy", "copy", 4, 2048, 16, 8, 128, "bf16", 0, 0, 777),
        # one sequence forked four ways (parallel sampling) and the old forks freed first: a few pages in one layer
        _pages("pages_fork_small", "fork", 1, 512, 16, 8, 128, "bf16", 1, 1003, 4),
        # beam search over a whole cache: 16 sequences, 64 forks, every layer's half-filled last pages copied
        _pages("pages_fork_beams", "fork", 4, 4224, 16, 8, 128, "bf16", 16, 4091, 64),
        # a pool with holes moved together, every layer
        _pages("pages_compact", "compact", 4, 4096, 16, 8, 128, "bf16", 48, 640, 0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    kind = rng.choice(["prefill", "prefill", "prefill", "shared", "shared", "pages"])
    while True:
        heads, kv_heads = rng.choice([(8, 2), (32, 8), (32, 8), (64, 8), (96, 12), (8, 8), (6, 1), (28, 4)])
        dim, dtype = rng.choice([64, 128, 128, 256]), rng.choice(["bf16", "bf16", "fp16"])
        page = rng.choice([1, 16, 16, 64, 48])
        fp8 = rng.random() < 0.3
        cap = rng.choice([0.0, 0.0, 0.0, 30.0])
        if kind == "prefill":
            form = rng.choice(["packed", "chunk", "drafts"])
            batch = _log(rng, 1, 24)
            if form == "packed":
                q = [_log(rng, 1, 8192) for _ in range(batch)]
                kv = list(q)
                page, fp8 = 0, False
            elif form == "chunk":
                q = [_log(rng, 16, 1024) for _ in range(batch)]
                kv = [n + _log(rng, 1, 16384) for n in q]
            else:
                q = [rng.randint(1, 9) for _ in range(batch)]
                kv = [n + _log(rng, 1, 16384) for n in q]
            case = _prefill("", " ".join(map(str, q)), " ".join(map(str, kv)), heads, kv_heads, dim, dtype, page, fp8,
                            rng.random() < 0.8, cap)
        elif kind == "shared":
            groups = rng.choice([1, 1, 2, 3, 4])
            members = [_log(rng, 1, 48) for _ in range(groups)]
            case = _shared("", " ".join(str(_log(rng, 64, 16384)) for _ in range(groups)), " ".join(map(str, members)),
                           " ".join(str(_log(rng, 1, 2048)) for _ in range(sum(members))), heads, kv_heads, dim, dtype,
                           page, fp8, cap)
        else:
            action = rng.choice(["copy", "fork", "fork", "compact"])
            layers, page = _log(rng, 1, 8), rng.choice([16, 16, 32, 64])
            kvh, dim = rng.choice([(8, 128), (2, 128), (8, 64), (1, 256)])
            if action == "copy":
                pages = _log(rng, 64, 2048)
                case = _pages("", "copy", layers, pages, page, kvh, dim, dtype, 0, 0, _log(rng, 1, pages // 2))
            elif action == "fork":
                rows, length = _log(rng, 1, 16), _log(rng, 1, 4096)
                count = rows * rng.randint(1, 4)
                per = -(-length // page)
                case = _pages("", "fork", layers, rows * per + count + rng.randint(0, 64), page, kvh, dim, dtype, rows,
                              length, count)
            else:
                rows, length = _log(rng, 2, 48), _log(rng, 16, 640)
                case = _pages("", "compact", layers, 2 * rows * -(-length // page) + rng.randint(0, 200), page, kvh, dim,
                              dtype, rows, length, 0)
        case.pop("name")
        w = work(case)
        if w["flops"] <= 1.0e12 and w["bytes"] <= 1.0e9 and _state_bytes(case) <= 4e9:
            return case


def _state_bytes(case):
    """Rough size of the inputs of a case."""
    if case["kind"] == "pages":
        return 2 * case["layers"] * case["pages"] * case["page"] * case["kv_heads"] * case["dim"] * 2
    tokens = sum(_ints(case["kv_lens"])) + sum(_ints(case.get("prefix_lens", "")))
    return 2 * tokens * case["kv_heads"] * case["dim"] * 2


def work(case):
    """Bytes: every input read once, every output written once.  Operations: the multiplications and additions of the two
    matrix products over the keys that a row sees (softmax not counted)."""
    if case["kind"] == "pages":
        return _pages_work(case)
    kv = _ints(case["kv_lens"])
    hq, hkv, d = case["heads"], case["kv_heads"], case["dim"]
    kv_item = 1 if case["fp8"] else 2
    if case["kind"] == "prefill":
        ql = _ints(case["q_lens"])
        rows = sum(ql)
        # keys seen by all rows of a sequence
        seen = sum(sum(range(n - q + 1, n + 1)) if case["causal"] else q * n for q, n in zip(ql, kv))
        tokens = sum(kv)
    else:
        pre, mem = _ints(case["prefix_lens"]), _ints(case["members"])
        rows = sum(mem)
        seen = sum(kv) + sum(p * m for p, m in zip(pre, mem))
        tokens = sum(kv) + sum(pre)
    byt = rows * hq * d * 2 * 2 + rows * hq * 4 + 2 * tokens * hkv * d * kv_item
    if case["page"]:
        byt += 4 * tokens // case["page"]
    return {"bytes": byt, "flops": 4 * d * hq * seen}


def _pages_work(case):
    row = case["kv_heads"] * case["dim"] * 2                     # bytes of one token's K (or V) row
    if case["action"] == "copy":
        return {"bytes": 2 * 2 * case["count"] * case["layers"] * case["page"] * row, "flops": 0}
    per = -(-case["length"] // case["page"])
    if case["action"] == "fork":
        part = case["length"] % case["page"]
        # the forks' tables are read for freeing, the parents' copied to them; the partial last pages move
        return {"bytes": 2 * 2 * case["count"] * case["layers"] * part * row + 3 * 4 * case["count"] * per
                + 4 * case["pages"], "flops": 0}
    moved, _, live = _compact_counts(case)
    return {"bytes": 2 * 2 * moved * case["layers"] * case["page"] * row + 2 * 4 * live + 2 * 4 * case["pages"], "flops": 0}


# ------------------------------------------------------------------------------------------------ inputs

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(gen, shape, dtype):
    return torch.randn(shape, generator=gen, device=DEV, dtype=dtype)


def _starts(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return torch.tensor(out, dtype=torch.int32, device=DEV)


def _fp8(gen, shape, heads):
    """e4m3 values of N(0, 1) numbers with a scale for each head, a few spare pages' worth of slack in the scale."""
    scale = torch.rand(heads, generator=gen, device=DEV) * 0.004 + 0.008
    x = torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32)
    return (x / scale.view(-1, 1)).clamp(-448.0, 448.0).to(torch.float8_e4m3fn), scale


def _pool(case, gen, lens_lists):
    """A pool with the pages of several tables in a shuffled order, eight pages to spare, and the tables."""
    P, hkv, d = case["page"], case["kv_heads"], case["dim"]
    need = [[-(-n // P) for n in lens] for lens in lens_lists]
    total = sum(map(sum, need)) + 8
    order = torch.randperm(total, generator=gen, device=DEV).to(torch.int32)
    tables, at = [], 0
    for counts in need:
        width = max(1, max(counts))
        table = torch.zeros((len(counts), width), dtype=torch.int32, device=DEV)
        for i, c in enumerate(counts):
            table[i, :c] = order[at:at + c]
            at += c
        tables.append(table)
    shape = (total, P, hkv, d)
    if case["fp8"]:
        k, ks = _fp8(gen, shape, hkv)
        v, vs = _fp8(gen, shape, hkv)
    else:
        k, v, ks, vs = _randn(gen, shape, DTYPES[case["dtype"]]), _randn(gen, shape, DTYPES[case["dtype"]]), None, None
    return k, v, ks, vs, tables


def prepare(case, seed):
    gen = _gen(seed)
    if case["kind"] == "pages":
        return _prepare_pages(case, gen)
    dt, d = DTYPES[case["dtype"]], case["dim"]
    kv = _ints(case["kv_lens"])
    s = {"case": case, "scale": d ** -0.5, "soft_cap": case["soft_cap"],
         "kv_lens": torch.tensor(kv, dtype=torch.int32, device=DEV)}
    if case["kind"] == "prefill":
        ql = _ints(case["q_lens"])
        s["q"] = _randn(gen, (sum(ql), case["heads"], d), dt)
        s["cu_q"], s["cu_k"] = _starts(ql), _starts(kv)
        if case["page"]:
            s["k"], s["v"], s["k_scale"], s["v_scale"], (s["table"],) = _pool(case, gen, [kv])
        else:
            s["k"], s["v"] = (_randn(gen, (sum(kv), case["kv_heads"], d), dt) for _ in range(2))
            s["k_scale"] = s["v_scale"] = s["table"] = None
    else:
        pre, mem = _ints(case["prefix_lens"]), _ints(case["members"])
        s["q"] = _randn(gen, (sum(mem), case["heads"], d), dt)
        s["k"], s["v"], s["k_scale"], s["v_scale"], (s["table"], s["prefix_table"]) = _pool(case, gen, [kv, pre])
        s["prefix_lens"] = torch.tensor(pre, dtype=torch.int32, device=DEV)
        s["group_starts"] = _starts(mem)
    return s


def _compact_counts(case):
    """The rows of a pool that is to be moved together were laid out round by round over the whole pool, and every other
    row has been freed since: (pages that move, tables' entries, live pages)."""
    live = _compact_tables(case)
    flat = [p for row in live for p in row]
    n = len(flat)
    return sum(1 for p in flat if p >= n), n, n


def _compact_tables(case):
    """Pages of the rows that are left.  The rows took pages in turn (every row one page a round, with lengths that fall
    by one page every third row), so holes are spread over the pool."""
    per = -(-case["length"] // case["page"])
    counts = [max(1, per - (r // 3) % max(1, per // 4 + 1)) for r in range(2 * case["rows"])]
    pages, nxt = [[] for _ in counts], 0
    for rnd in range(max(counts)):
        for r, c in enumerate(counts):
            if rnd < c:
                pages[r].append(nxt)
                nxt += 1
    return pages[1::2]


def _prepare_pages(case, gen):
    dt = DTYPES[case["dtype"]]
    shape = (case["layers"], case["pages"], case["page"], case["kv_heads"], case["dim"])
    s = {"case": case, "k": _randn(gen, shape, dt), "v": _randn(gen, shape, dt)}
    if case["action"] == "copy":
        order = torch.randperm(case["pages"], generator=gen, device=DEV).to(torch.int32)
        s["src"], s["dst"] = order[:case["count"]].clone(), order[-case["count"]:].clone()
        return s
    refs = torch.zeros(case["pages"], dtype=torch.int32)
    if case["action"] == "fork":
        # rows 0 .. rows - 1 are the parents; the forks behind them hold last step's forks, which are freed first
        rows, count, length, page = case["rows"], case["count"], case["length"], case["page"]
        per = -(-length // page)
        order = torch.randperm(case["pages"], generator=gen, device=DEV).to(torch.int32).cpu()
        table = torch.full((rows + count, per + 2), -1, dtype=torch.int32)
        table[:rows, :per] = order[:rows * per].view(rows, per)
        refs[order[:rows * per].long()] = 1
        parents = torch.arange(count) % rows
        spare = order[rows * per:].sort().values
        for i, p in enumerate(parents.tolist()):
            table[rows + i, :per] = table[p, :per]
            if length % page:
                table[rows + i, per - 1] = spare[i]
                refs[spare[i]] = 1
                refs[table[p, :per - 1].long()] += 1
            else:
                refs[table[p, :per].long()] += 1
        s["parents"] = parents.to(torch.int32).to(DEV)
        s["children"] = (torch.arange(count) + rows).to(torch.int32).to(DEV)
        s["lens"] = torch.full((rows + count,), length, dtype=torch.int32, device=DEV)
    else:
        live = _compact_tables(case)
        table = torch.full((len(live), max(map(len, live))), -1, dtype=torch.int32)
        for r, pages in enumerate(live):
            table[r, :len(pages)] = torch.tensor(pages, dtype=torch.int32)
            refs[torch.tensor(pages)] = 1
        s["lens"] = torch.tensor([len(p) * case["page"] - r % case["page"] for r, p in enumerate(live)], dtype=torch.int32,
                                 device=DEV)
        s["table0"], s["refs0"] = table.to(DEV), refs.to(DEV)
    s["table"], s["refs"] = table.to(DEV), refs.to(DEV)
    return s


# ------------------------------------------------------------------------------------------------ one pass

def run(state):
    kind = state["case"]["kind"]
    if own:
        return _own(kind, state)
    if kind == "prefill":
        return _plain_prefill(state)
    if kind == "shared":
        return _plain_shared(state)
    return _plain_pages(state)


def _own(kind, s):
    import triton_dist_amd as fd
    case = s["case"]
    if kind == "prefill":
        lse = torch.empty(s["q"].shape[0], case["heads"], dtype=torch.float32, device=DEV)
        paged = s["table"] is not None
        out = fd.gqa_fwd_batch_prefill(s["q"], s["k"], s["v"], s["cu_q"], s["kv_lens"] if paged else None, s["table"],
                                       s["scale"], s["soft_cap"], causal=case["causal"],
                                       cu_seqlens_k=None if paged else s["cu_k"], lse_out=lse, k_scale=s["k_scale"],
                                       v_scale=s["v_scale"])
        return {"out": out, "lse": lse}
    if kind == "shared":
        lse = torch.empty(s["q"].shape[0], case["heads"], dtype=torch.float32, device=DEV)
        out = fd.gqa_fwd_batch_decode_shared_prefix(
            s["q"], s["k"], s["v"], None, [1] * s["q"].shape[0], s["kv_lens"], s["table"], s["prefix_lens"],
            s["prefix_table"], s["scale"], s["soft_cap"], group_starts=s["group_starts"], lse_out=lse,
            k_scale=s["k_scale"], v_scale=s["v_scale"])
        return {"out": out, "lse": lse}
    if case["action"] == "copy":
        fd.paged_kv_copy(s["k"], s["v"], s["src"], s["dst"])
        return {"k": s["k"], "v": s["v"]}
    if case["action"] == "fork":
        fd.paged_kv_free(s["table"], s["lens"], s["refs"], s["children"])
        ok = fd.paged_kv_fork(s["k"], s["v"], s["table"], s["lens"], s["refs"], s["parents"], s["children"])
        return {"k": s["k"], "v": s["v"], "table": s["table"], "lens": s["lens"], "refs": s["refs"], "ok": ok}
    s["table"].copy_(s["table0"])          # the pool as it was: the pages that move are where they were
    s["refs"].copy_(s["refs0"])
    live = fd.paged_kv_compact(s["k"], s["v"], s["table"], s["refs"])
    return {"k": s["k"], "v": s["v"], "table": s["table"], "refs": s["refs"], "live": live}


def _attend(q, k, v, visible, scale, soft_cap):
    """q [T, H, D], k and v [N, Hkv, D] in 32 bits; visible [T]: how many keys a row sees -> out [T, H, D], lse [T, H]."""
    T, H, D = q.shape
    N, hkv, _ = k.shape
    G = H // hkv
    kt, vt = k.permute(1, 2, 0).contiguous(), v.permute(1, 0, 2).contiguous()      # [Hkv, D, N], [Hkv, N, D]
    out = torch.empty(T, H, D, dtype=torch.float32, device=q.device)
    lse = torch.empty(T, H, dtype=torch.float32, device=q.device)
    step = max(1, ROWS_AT_ONCE // G)
    for t0 in range(0, T, step):
        t1 = min(T, t0 + step)
        rows = q[t0:t1].reshape(t1 - t0, hkv, G, D).permute(1, 0, 2, 3).reshape(hkv, (t1 - t0) * G, D)
        x = torch.bmm(rows, kt) * scale                                             # [Hkv, rows, N]
        if soft_cap > 0:
            x = soft_cap * torch.tanh(x / soft_cap)
        seen = torch.arange(N, device=q.device)[None, :] < visible[t0:t1].repeat_interleave(G)[:, None]
        x = torch.where(seen[None], x, torch.full((), float("-inf"), device=q.device))
        m = x.amax(-1, keepdim=True) if N else torch.full((hkv, x.shape[1], 1), float("-inf"), device=q.device)
        m0 = torch.where(m > float("-inf"), m, torch.zeros_like(m))
        p = torch.exp(x - m0)
        total = p.sum(-1, keepdim=True)
        o = torch.bmm(p, vt) / torch.where(total > 0, total, torch.ones_like(total))
        ls = torch.where(total > 0, m0 + torch.log(total), torch.full_like(total, float("-inf")))
        out[t0:t1] = o.reshape(hkv, t1 - t0, G, D).permute(1, 0, 2, 3).reshape(t1 - t0, H, D)
        lse[t0:t1] = ls.reshape(hkv, t1 - t0, G).permute(1, 0, 2).reshape(t1 - t0, H)
    return out, lse


def _rows_of(pool, table_row, n, scale):
    """The first n tokens of a sequence, [n, Hkv, D] in 32 bits."""
    P = pool.shape[1]
    x = pool[table_row[:-(-n // P)].long()].reshape(-1, pool.shape[2], pool.shape[3])[:n].float()
    return x if scale is None else x * scale[None, :, None]


def _plain_prefill(s):
    case = s["case"]
    out = torch.empty_like(s["q"])
    lse = torch.empty(s["q"].shape[:2], dtype=torch.float32, device=DEV)
    at, ak = 0, 0
    for b, (n, nk) in enumerate(zip(_ints(case["q_lens"]), _ints(case["kv_lens"]))):
        if s["table"] is None:
            k, v = s["k"][ak:ak + nk].float(), s["v"][ak:ak + nk].float()
        else:
            k = _rows_of(s["k"], s["table"][b], nk, s["k_scale"])
            v = _rows_of(s["v"], s["table"][b], nk, s["v_scale"])
        pos = torch.arange(n, device=DEV)
        visible = pos + (nk - n + 1) if case["causal"] else torch.full_like(pos, nk)
        o, ls = _attend(s["q"][at:at + n].float(), k, v, visible, s["scale"], s["soft_cap"])
        out[at:at + n], lse[at:at + n] = o.to(out.dtype), ls
        at, ak = at + n, ak + nk
    return {"out": out, "lse": lse}


def _plain_shared(s):
    case = s["case"]
    out = torch.empty_like(s["q"])
    lse = torch.empty(s["q"].shape[:2], dtype=torch.float32, device=DEV)
    kv, b = _ints(case["kv_lens"]), 0
    for g, (pre, members) in enumerate(zip(_ints(case["prefix_lens"]), _ints(case["members"]))):
        kp = _rows_of(s["k"], s["prefix_table"][g], pre, s["k_scale"])
        vp = _rows_of(s["v"], s["prefix_table"][g], pre, s["v_scale"])
        for _ in range(members):
            k = torch.cat((kp, _rows_of(s["k"], s["table"][b], kv[b], s["k_scale"])))
            v = torch.cat((vp, _rows_of(s["v"], s["table"][b], kv[b], s["v_scale"])))
            o, ls = _attend(s["q"][b:b + 1].float(), k, v, torch.tensor([pre + kv[b]], device=DEV), s["scale"],
                            s["soft_cap"])
            out[b], lse[b] = o[0].to(out.dtype), ls[0]
            b += 1
    return {"out": out, "lse": lse}


def _plain_pages(s):
    case = s["case"]
    k, v = s["k"], s["v"]
    if case["action"] == "copy":
        src, dst = s["src"].long(), s["dst"].long()
        k[:, dst] = k[:, src]
        v[:, dst] = v[:, src]
        return {"k": k, "v": v}
    if case["action"] == "fork":
        table, lens, refs, P = s["table"], s["lens"], s["refs"], case["page"]
        rows = s["children"].long()
        old = table[rows]
        refs.index_add_(0, old[old >= 0].long(), torch.full((int((old >= 0).sum()),), -1, dtype=torch.int32, device=DEV))
        table[rows] = -1
        lens[rows] = 0
        parents = s["parents"].long()
        n = lens[parents]
        whole, part = n // P, n % P
        width = torch.arange(table.shape[1], device=DEV)[None, :]
        new = torch.where(width < whole[:, None], table[parents], torch.full_like(table[parents], -1))
        wants = (part > 0).nonzero()[:, 0]
        fresh = (refs == 0).nonzero()[:wants.numel(), 0]
        ok = torch.ones_like(s["children"])
        ok[wants[fresh.numel():]] = 0
        wants = wants[:fresh.numel()]
        new[wants, whole[wants].long()] = fresh.to(torch.int32)
        new = torch.where(ok[:, None] > 0, new, torch.full_like(new, -1))
        table[rows] = new
        lens[rows] = torch.where(ok > 0, n, torch.zeros_like(n))
        refs.index_add_(0, new[new >= 0].long(), torch.ones(int((new >= 0).sum()), dtype=torch.int32, device=DEV))
        if wants.numel():
            last = table[parents[wants], whole[wants].long()].long()
            tok = torch.arange(P, device=DEV)[None, :] < part[wants][:, None]          # [wants, P]
            for pool in (k, v):
                pool[:, fresh] = torch.where(tok[None, :, :, None, None], pool[:, last], pool[:, fresh])
        return {"k": k, "v": v, "table": table, "lens": lens, "refs": refs, "ok": ok}
    s["table"].copy_(s["table0"])
    s["refs"].copy_(s["refs0"])
    table, refs = s["table"], s["refs"]
    live = (refs > 0).sum().to(torch.int32).view(1)
    ids = torch.arange(refs.numel(), device=DEV)
    src, dst = ((refs > 0) & (ids >= live)).nonzero()[:, 0], ((refs == 0) & (ids < live)).nonzero()[:, 0]
    k[:, dst] = k[:, src]
    v[:, dst] = v[:, src]
    refs[dst] = refs[src]
    refs[src] = 0
    to = ids.to(torch.int32)
    to[src] = dst.to(torch.int32)
    table.copy_(torch.where(table >= 0, to[table.clamp_min(0).long()], table))
    return {"k": k, "v": v, "table": table, "refs": refs, "live": live}


# ------------------------------------------------------------------------------------------------ 64 bits

def exact(case, seed):
    """Attention from its definition, one head and a slab of rows at a time, in 64 bits; pages hold no computed numbers."""
    if case["kind"] == "pages":
        return None
    s = prepare(case, seed)
    H, D, hkv = case["heads"], case["dim"], case["kv_heads"]
    kv = _ints(case["kv_lens"])

    def gather(pool, tab, n, scale, h):
        idx = torch.arange(n, device=DEV)
        x = pool[tab[idx // pool.shape[1]].long(), idx % pool.shape[1], h].double()
        return x if scale is None else x * scale[h].double()

    jobs = []          # (first row, rows, keys of a head, first row's keys, growth of the keys from row to row)
    if case["kind"] == "prefill":
        at, ak = 0, 0
        for b, (n, nk) in enumerate(zip(_ints(case["q_lens"]), kv)):
            if s["table"] is None:
                keys = lambda h, a=ak, m=nk: (s["k"][a:a + m, h].double(), s["v"][a:a + m, h].double())  # noqa: E731
            else:
                keys = lambda h, i=b, m=nk: (gather(s["k"], s["table"][i], m, s["k_scale"], h),            # noqa: E731
                                             gather(s["v"], s["table"][i], m, s["v_scale"], h))
            jobs.append((at, n, keys, nk - n + 1 if case["causal"] else nk, 1 if case["causal"] else 0))
            at, ak = at + n, ak + nk
    else:
        b = 0
        for g, (pre, members) in enumerate(zip(_ints(case["prefix_lens"]), _ints(case["members"]))):
            for _ in range(members):
                def keys(h, i=b, j=g, m=kv[b], p=pre):
                    return tuple(torch.cat((gather(s[c], s["prefix_table"][j], p, s[c + "_scale"], h),
                                            gather(s[c], s["table"][i], m, s[c + "_scale"], h))) for c in ("k", "v"))
                jobs.append((b, 1, keys, pre + kv[b], 0))
                b += 1
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    lse = torch.full(s["q"].shape[:2], float("-inf"), dtype=torch.float64, device=DEV)
    for at, n, keys, first, growth in jobs:
        for hk in range(hkv):
            k, v = keys(hk)
            for h in range(hk * (H // hkv), (hk + 1) * (H // hkv)):
                for r0 in range(0, n, 4096):
                    r1 = min(n, r0 + 4096)
                    x = (s["q"][at + r0:at + r1, h].double() @ k.t()) * s["scale"]
                    if case["soft_cap"] > 0:
                        x = torch.tanh(x / case["soft_cap"]) * case["soft_cap"]
                    if growth:
                        limit = first + torch.arange(r0, r1, device=DEV)
                        x.masked_fill_(torch.arange(k.shape[0], device=DEV)[None, :] >= limit[:, None], float("-inf"))
                    total = torch.logsumexp(x, -1)
                    w = torch.exp(x - torch.where(total > float("-inf"), total, torch.zeros_like(total))[:, None])
                    out[at + r0:at + r1, h] = w @ v
                    lse[at + r0:at + r1, h] = total
    return {"out": out, "lse": lse}
