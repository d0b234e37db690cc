"""The scored-attention and 8-bit cache operators as they are called, case by case.

Four operators of the pooled KV cache and the attention that reads it:

  append8   new K and V rows into pages of 8-bit codes with one scale for each page and head
  attend    attention over pages of 8-bit codes (decode, verify, a prompt chunk) ...
            ... and over bf16 rows, with scores capped by a tanh, a distance bias, a sliding window,
            packed documents or a bidirectional prefix
  pages     copies of whole or partial pages in every layer's pool: forks that write, compaction

`listed()` and `draw()` describe calls, `prepare()` makes what a program has in hand before one, `run()` is the
call (plain torch operations, or the library's kernels when `own` is true), `exact()` its answer in 64 bits.
"""
import ctypes as C
import math

import numpy as np
import torch

own = False
DEV = "cuda"
LIMIT = {"e4m3": 448.0, "i8": 127.0}


# ---- the cases ------------------------------------------------------------------------------------


def _attend(name=None, **fields):
    case = dict(kind="attend", sessions=1, rows=1, heads=32, kv_heads=8, dim=128, low=1, high=1, cache="bf16", page=0,
                causal=True, cap=0.0, bias=False, window=0, mask="none", documents=0, prefix=0)
    case.update(fields)
    return dict(case, name=name) if name else case


def _append(name=None, **fields):
    case = dict(kind="append8", sessions=1, rows=1, kv_heads=8, dim=128, low=0, high=0, cache="e4m3", page=64)
    case.update(fields)
    return dict(case, name=name) if name else case


def _pages(name=None, **fields):
    case = dict(kind="pages", pools=64, blocks=96, page=64, row_bytes=1024, copies=32, whole=False)
    case.update(fields)
    return dict(case, name=name) if name else case


def listed():
    return [
        # one decode step of a batch writes one row for each session: latency
        _append("append8_step", sessions=64, rows=1, low=1, high=2047),
        # four prompts enter the cache behind a short shared beginning that ends inside a page
        _append("append8_prompts", sessions=4, rows=4093, low=37, high=37, cache="i8"),
        # one token of one chat session: the smallest call of the attention
        _attend("decode8_single", low=4096, high=4096, cache="e4m3", page=64),
        # a full batch of sessions of very different lengths: the cache is read once, nothing else counts
        _attend("decode8_batch", sessions=64, heads=40, low=512, high=32768, cache="e4m3", page=64),
        # four drafted tokens verified over one long history in small pages, scores capped
        _attend("verify8_long", rows=4, low=131072, high=131072, cache="i8", page=16, cap=30.0),
        # a chunk of a prompt over the history that the cache already holds
        _attend("chunk8_prompt", rows=2048, low=16384, high=16384, cache="e4m3", page=64),
        # a batch's decode step in a layer with capped scores and a sliding window
        _attend("capped_window_decode", sessions=64, heads=40, low=512, high=32768, page=64, cap=50.0, window=4096),
        # two long prompts in a layer whose scores are capped: the largest call
        _attend("capped_prompts", sessions=2, rows=8192, heads=40, low=8192, high=8192, cap=50.0),
        # many short documents packed into one sequence, each with a bias that depends on distance
        _attend("packed_documents", rows=16384, low=16384, high=16384, mask="documents", documents=2048, bias=True),
        # prompts of an odd length whose first part (an image, an instruction) is seen from both sides
        _attend("prefix_prompts", sessions=4, rows=1531, heads=40, low=1531, high=1531, mask="prefix", prefix=700,
                cap=30.0),
        # forked sessions are about to write: their last, partly filled pages become their own in every layer
        _pages("fork_pages", pools=64, blocks=96, copies=32),
        # a pool is compacted after many sessions have ended: whole pages move to the front
        _pages("compact_pages", pools=16, blocks=1536, copies=700, whole=True),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["append8", "attend8", "attend8", "decode", "prompt", "prompt", "pages"])
    if kind == "append8":
        sessions = _spread(rng, 1, 64)
        return _append(sessions=sessions, rows=_spread(rng, 1, max(1, 16384 // sessions)), kv_heads=rng.choice([1, 2, 4, 8, 16]),
                       low=rng.randint(0, 100), high=rng.randint(100, 700), cache=rng.choice(["e4m3", "i8"]),
                       page=rng.choice([16, 32, 64, 128]))
    if kind == "pages":
        copies = _spread(rng, 1, 700)
        return _pages(pools=_spread(rng, 1, 64), blocks=2 * copies + rng.randint(0, 64), copies=copies,
                      page=rng.choice([16, 32, 64]), row_bytes=rng.choice([256, 512, 1024]), whole=rng.random() < 0.5)
    kv_heads = rng.choice([1, 2, 4, 8, 16])
    score = dict(kv_heads=kv_heads, heads=kv_heads * rng.choice([1, 2, 4, 5, 8]), cap=rng.choice([0.0, 20.0, 30.0, 50.0]),
                 bias=rng.random() < 0.4)
    if kind in ("attend8", "decode"):
        sessions = _spread(rng, 1, 96)
        rows = rng.choice([1, 1, 1, 2, 3, 4, 8])
        high = _spread(rng, 16, max(16, min(65536, 6000000 // (sessions * kv_heads))))
        cache = rng.choice(["e4m3", "i8"]) if kind == "attend8" else "bf16"
        page = rng.choice([16, 32, 64, 128]) if kind == "attend8" else rng.choice([0, 64, 128])
        return _attend(sessions=sessions, rows=rows, low=rng.randint(max(1, high // 8), high), high=high, cache=cache, page=page,
                       window=rng.choice([0, 0, 0, 1024, 4096]), **score)
    rows, sessions = _spread(rng, 100, 6000), rng.choice([1, 1, 2, 3])
    mask = rng.choice(["none", "documents", "prefix"])
    coded = mask == "none" and rng.random() < 0.3
    before = rng.randint(0, 4000) if mask == "none" else 0
    rows = min(rows, 2000000000 // (sessions * score["heads"] * (rows + before)))
    return _attend(sessions=sessions, rows=rows, low=rows + before,
                   high=0, cache=rng.choice(["e4m3", "i8"]) if coded else "bf16", page=64 if coded else 0, mask=mask,
                   documents=rng.randint(50, 1500), prefix=rng.randint(1, rows),
                   causal=mask != "none" or rng.random() < 0.8, window=rng.choice([0, 0, 1000]) if mask == "none" else 0, **score)


# ---- geometry -------------------------------------------------------------------------------------


def _lengths(case):
    """Rows in the cache, session by session: the ends of the range and, between them, an even spread out of order."""
    low, n = case["low"], case["sessions"]
    high = max(low, case["high"])
    if n == 1:
        return [high]
    between = [low + int((high - low) * ((i * 0.6180339887) % 1.0)) for i in range(n - 2)]
    return [high] + between + [low]


def _documents(case):
    """The packed documents of a sequence: (start, end) until its rows are used up."""
    out, at, i = [], 0, 0
    while at < case["rows"]:
        n = 1 + int(2 * case["documents"] * ((0.381966 + i * 0.6180339887) % 1.0))
        out.append((at, min(case["rows"], at + n)))
        at, i = at + n, i + 1
    return out


def _ranges(case):
    """[first, end) of the tokens each row sees, int32 [sessions][rows]; and each row's own position."""
    lengths = np.array(_lengths(case))[:, None]
    row = np.arange(case["rows"])[None, :]
    position = lengths - case["rows"] + row
    first = np.zeros_like(position)
    end = position + 1 if case["causal"] else np.broadcast_to(lengths, position.shape).copy()
    if case["window"]:
        first = np.maximum(first, position + 1 - case["window"])
    if case["mask"] == "documents":
        for start, _ in _documents(case):
            first[:, start:] = start
    if case["mask"] == "prefix":
        for b in range(case["sessions"]):
            end[b] = np.maximum(end[b], max(1, case["prefix"] - 61 * b))
    return np.clip(first, 0, lengths).astype(np.int32), np.clip(end, 0, lengths).astype(np.int32), position


def work(case):
    if case["kind"] == "append8":
        elements = 2 * case["sessions"] * case["rows"] * case["kv_heads"] * case["dim"]
        touched = sum(-(-(n + case["rows"]) // case["page"]) - n // case["page"] for n in _lengths(case))
        return {"bytes": 3 * elements + 8 * touched * case["kv_heads"], "flops": 2 * elements}
    if case["kind"] == "pages":
        moved = sum(_page_rows(case)) * case["row_bytes"] * case["pools"]
        return {"bytes": 2 * moved, "flops": 0}
    first, end, _ = _ranges(case)
    first, end = first.astype(np.int64), end.astype(np.int64)
    pairs = int(np.maximum(end - first, 0).sum())
    tokens = int((end.max(1) - first.min(1)).sum())
    width = case["kv_heads"] * case["dim"]
    moved = 4 * case["sessions"] * case["rows"] * case["heads"] * case["dim"]
    if case["cache"] == "bf16":
        moved += 4 * tokens * width
    else:
        moved += 2 * tokens * width + 8 * (tokens // case["page"] + 1) * case["kv_heads"]
    return {"bytes": moved, "flops": 4 * pairs * case["heads"] * case["dim"]}


# ---- inputs ---------------------------------------------------------------------------------------


def _generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _loud(x):
    """Keys as projections publish them: a few channels are several times louder than the others."""
    x[..., 5::32] *= 3.0
    return x


def _power_scale(amax, limit):
    """The smallest power of two s >= 2^-126 with amax <= limit * s."""
    _, e = torch.frexp(amax)
    s = torch.ldexp(torch.ones_like(amax), (e - 1 - math.frexp(limit)[1] + 1).clamp(min=-126))
    return torch.where(amax == 0, 2.0 ** -126, torch.where(amax > limit * s, 2 * s, s))


def _encode(x, cache):
    return x.to(torch.float8_e4m3fn) if cache == "e4m3" else torch.round(x).to(torch.int8)


def _pool8(case, g, pages, loud):
    """A pool of full pages: codes [page][head][token][dim] and scales [page][head]."""
    codes, scales = [], []
    for at in range(0, pages, 512):
        x = _normal(g, min(512, pages - at), case["kv_heads"], case["page"], case["dim"])
        x = (_loud(x) if loud else x) * torch.exp(0.5 * _normal(g, x.shape[0], case["kv_heads"], 1, 1))
        s = _power_scale(x.abs().amax((2, 3)), LIMIT[case["cache"]])
        codes.append(_encode(x / s[:, :, None, None], case["cache"]))
        scales.append(s)
    return torch.cat(codes), torch.cat(scales)


def _table(case, g, lengths):
    """Pages in no order; -1 behind a session's last."""
    need = [-(-n // case["page"]) for n in lengths]
    order = torch.randperm(sum(need) + 3, generator=g, device=DEV).to(torch.int32)
    table = torch.full((len(need), max(1, max(need))), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, int(order.numel())


def _inputs(case, seed):
    g = _generator(seed)
    s = {"case": case}
    if case["kind"] == "append8":
        before = _lengths(case)
        s["before"] = before
        s["table"], blocks = _table(case, g, [n + case["rows"] for n in before])
        for x in ("k", "v"):
            new = _normal(g, case["sessions"], case["rows"], case["kv_heads"], case["dim"])
            s[x] = ((_loud(new) if x == "k" else new) * 1.5).to(torch.bfloat16)
            s[x + "_codes"], s[x + "_scales"] = _pool8(case, g, blocks, x == "k")
        s["kv_tokens"] = torch.tensor(before, dtype=torch.int32, device=DEV)
        return s
    if case["kind"] == "pages":
        shape = (case["blocks"], case["page"], case["row_bytes"])
        s["pools"] = [torch.randint(-128, 128, shape, dtype=torch.int8, generator=g, device=DEV) for _ in range(case["pools"])]
        order = torch.randperm(case["blocks"], generator=g, device=DEV).cpu().tolist()
        n, rows = case["copies"], _page_rows(case)
        # a fork copies one page to several children; a compaction moves each page once
        sources = order[n:2 * n] if case["whole"] else [order[n + i // 4] for i in range(n)]
        s["moves"] = [(a, b, r) for a, b, r in zip(sources, order[:n], rows)]
        return s
    lengths = _lengths(case)
    s["lengths"] = lengths
    s["kv_tokens"] = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    s["q"] = (3.0 * _normal(g, case["sessions"], case["rows"], case["heads"], case["dim"])).to(torch.bfloat16)
    if case["bias"]:
        s["slopes"] = torch.exp2(-8.0 * (1 + torch.arange(case["heads"], device=DEV, dtype=torch.float32)) / case["heads"])
    if case["cache"] != "bf16":
        s["table"], blocks = _table(case, g, lengths)
        for x in ("k", "v"):
            s[x], s[x + "_scales"] = _pool8(case, g, blocks, x == "k")
            tail = s[x].view(torch.int8)
            for b, n in enumerate(lengths):    # what lies behind the last token may be anything
                if n % case["page"]:
                    tail[s["table"][b, n // case["page"]], :, n % case["page"]:] = 127
    else:
        if case["page"]:
            s["table"], blocks = _table(case, g, lengths)
            shape = (blocks, case["page"], case["kv_heads"], case["dim"])
        else:
            shape = (case["sessions"], max(lengths), case["kv_heads"], case["dim"])
        s["k"], s["v"] = _loud(_normal(g, *shape)).to(torch.bfloat16), _normal(g, *shape).to(torch.bfloat16)
    if case["mask"] != "none":
        first, end, _ = _ranges(case)
        s["first"], s["end"] = torch.from_numpy(first).to(DEV), torch.from_numpy(end).to(DEV)
    return s


def _page_rows(case):
    n = case["copies"]
    return [case["page"] if case["whole"] else 1 + int((case["page"] - 1) * ((i * 0.6180339887) % 1.0)) for i in range(n)]


# ---- the plain forms ------------------------------------------------------------------------------


def _session_rows(s, x, b, dtype):
    """K or V of one session as [kv_heads][token][dim]."""
    case, n = s["case"], s["lengths"][b]
    if not case["page"]:
        return s[x][b, :n].to(dtype).permute(1, 0, 2)
    pages = s["table"][b, :-(-n // case["page"])].long()
    if case["cache"] == "bf16":
        return s[x][pages].to(dtype).flatten(0, 1)[:n].permute(1, 0, 2)
    rows = s[x][pages].to(dtype) * s[x + "_scales"][pages].to(dtype)[:, :, None, None]
    return rows.permute(1, 0, 2, 3).flatten(1, 2)[:, :n]


def _plain_attend(s):
    case = s["case"]
    group, rows = case["heads"] // case["kv_heads"], case["rows"]
    out = torch.zeros_like(s["q"])
    for b, n in enumerate(s["lengths"]):
        if not n:
            continue
        k, v = _session_rows(s, "k", b, torch.float32), _session_rows(s, "v", b, torch.float32)
        position = torch.arange(n - rows, n, device=DEV)[:, None]
        token = torch.arange(n, device=DEV)[None, :]
        if case["mask"] == "none":
            seen = token <= position if case["causal"] else torch.ones_like(token <= position)
            if case["window"]:
                seen = seen & (token > position - case["window"])
        else:
            seen = (token >= s["first"][b][:, None]) & (token < s["end"][b][:, None])
        distance = (position - token).abs().float() if case["bias"] else None
        step = max(1, min(case["kv_heads"], (1 << 30) // (group * rows * n)))
        for h in range(0, case["kv_heads"], step):
            kv = min(step, case["kv_heads"] - h)
            q = s["q"][b, :, h * group:(h + kv) * group].float().permute(1, 0, 2).reshape(kv, group * rows, case["dim"])
            score = (q @ k[h:h + kv].transpose(1, 2) / math.sqrt(case["dim"])).view(kv, group, rows, n)
            if case["cap"]:
                score = case["cap"] * torch.tanh(score / case["cap"])
            if case["bias"]:
                score = score - s["slopes"].view(-1, group)[h:h + kv, :, None, None] * distance
            score = score.masked_fill(~seen, -math.inf)
            top = score.amax(-1, keepdim=True)
            weight = torch.exp(score - torch.where(torch.isinf(top), 0.0, top))
            total = weight.sum(-1, keepdim=True)
            weight = weight / torch.where(total == 0, 1.0, total)
            got = (weight.view(kv, group * rows, n) @ v[h:h + kv]).view(kv * group, rows, case["dim"])
            out[b, :, h * group:(h + kv) * group] = got.permute(1, 0, 2).to(out.dtype)
    return out


def _plain_append(s):
    case = s["case"]
    page, rows = case["page"], case["rows"]
    blocks, start, owner = [], [], []
    for b, n in enumerate(s["before"]):
        for j in range(n // page, -(-(n + rows) // page)):
            blocks.append((b, j))
            start.append(j * page - n)             # the page's first slot, counted from the first new row
            owner.append(b)
    at = torch.tensor(blocks, device=DEV)
    block = s["table"][at[:, 0], at[:, 1]].long()
    owner = torch.tensor(owner, device=DEV)
    source = torch.tensor(start, device=DEV)[:, None] + torch.arange(page, device=DEV)[None, :]
    new, old = (source >= 0) & (source < rows), source < 0
    limit = LIMIT[case["cache"]]
    out = []
    for x in ("k", "v"):
        codes, scales = s[x + "_codes"], s[x + "_scales"]
        value = s[x][owner[:, None], source.clamp(0, rows - 1)].float().permute(0, 2, 1, 3)   # [page][head][slot][dim]
        amax = torch.where(new[:, None, :, None], value.abs(), 0.0).amax((2, 3))
        fresh = _power_scale(amax, limit)
        held = scales[block]
        fresh = torch.where(old.any(1)[:, None], torch.maximum(held, fresh), fresh)
        kept = codes[block].float() * (held / fresh)[:, :, None, None]
        kept = torch.where(old[:, None, :, None], _encode(kept, case["cache"]).float(), codes[block].float())
        value = torch.where(new[:, None, :, None], _encode(value / fresh[:, :, None, None], case["cache"]).float(), kept)
        codes[block] = value.to(codes.dtype)
        scales[block] = fresh
        out += [codes, scales]
    return out


def _plain_pages(s):
    source = torch.tensor([m[0] for m in s["moves"]], device=DEV)
    target = torch.tensor([m[1] for m in s["moves"]], device=DEV)
    rows = torch.tensor([m[2] for m in s["moves"]], device=DEV)
    moved = (torch.arange(s["case"]["page"], device=DEV)[None, :] < rows[:, None])[:, :, None]
    for pool in s["pools"]:
        pool[target] = torch.where(moved, pool[source], pool[target])
    return s["pools"]


# ---- the library's calls --------------------------------------------------------------------------


def _handle(s):
    """What a program keeps beside its buffers: the call's description with its plan, workspace and status word."""
    from clori_b200 import abi
    case, lib = s["case"], abi.load()
    s["lib"], s["status"] = lib, torch.zeros(1, dtype=torch.int32, device=DEV)
    if case["kind"] == "pages":
        a = abi.KvPagesArgs()
        pools = (abi.KvPagePool * case["pools"])()
        for pool, t in zip(pools, s["pools"]):
            pool.base, pool.blocks, pool.block_stride = t.data_ptr(), case["blocks"], case["page"] * case["row_bytes"]
            pool.segments, pool.row_bytes = 1, case["row_bytes"]
        moves = (abi.KvCopy * case["copies"])(*[(1, a_, b_, r) for a_, b_, r in s["moves"]])
        a.pools, a.pool_count, a.copies, a.copy_count, a.block_tokens = pools, case["pools"], moves, case["copies"], case["page"]
        s["args"], s["keep"] = a, (pools, moves)
        return
    codes = {"bf16": abi.KV_PLAIN, "e4m3": abi.KV_E4M3, "i8": abi.KV_I8}[case["cache"]]
    width, page = case["kv_heads"] * case["dim"], case["page"]
    if case["kind"] == "append8":
        a = abi.Kv8AppendArgs()
        a.sessions, a.tokens, a.kv_heads, a.head_dim, a.code = case["sessions"], case["rows"], case["kv_heads"], case["dim"], codes
        a.key, a.value, a.dtype = s["k"].data_ptr(), s["v"].data_ptr(), abi.DTYPE_BF16
        a.token_stride, a.session_stride = width, case["rows"] * width
        a.kv_tokens, a.block_table = s["kv_tokens"].data_ptr(), s["table"].data_ptr()
        a.block_tokens, a.block_table_stride, a.pool_blocks = page, s["table"].shape[1], s["k_codes"].shape[0]
        a.key_codes, a.value_codes = s["k_codes"].data_ptr(), s["v_codes"].data_ptr()
        a.code_token_stride, a.code_head_stride, a.code_block_stride = case["dim"], page * case["dim"], page * width
        a.key_scales, a.value_scales, a.scale_block_stride = s["k_scales"].data_ptr(), s["v_scales"].data_ptr(), case["kv_heads"]
        a.status = s["status"].data_ptr()
        s["args"] = a
        return
    p = abi.ScoredProblem()
    p.sessions, p.query_rows, p.query_heads, p.kv_heads, p.head_dim = (
        case["sessions"], case["rows"], case["heads"], case["kv_heads"], case["dim"])
    p.causal, p.scale, p.cap, p.window = int(case["causal"]), 1.0 / math.sqrt(case["dim"]), case["cap"], case["window"]
    p.query_dtype = p.output_dtype = abi.DTYPE_BF16
    p.kv_dtype, p.kv_code = abi.DTYPE_BF16 if case["cache"] == "bf16" else abi.DTYPE_I8, codes
    s["out"] = torch.empty_like(s["q"])
    p.query, p.output = s["q"].data_ptr(), s["out"].data_ptr()
    p.query_row_stride = case["heads"] * case["dim"]
    p.query_session_stride = case["rows"] * p.query_row_stride
    p.key, p.value = s["k"].data_ptr(), s["v"].data_ptr()
    if case["cache"] == "bf16":
        p.key_token_stride = p.value_token_stride = width
        p.key_head_stride = p.value_head_stride = case["dim"]
        p.key_outer_stride = p.value_outer_stride = s["k"].shape[1] * width
    else:
        p.key_token_stride = p.value_token_stride = case["dim"]
        p.key_head_stride = p.value_head_stride = page * case["dim"]
        p.key_outer_stride = p.value_outer_stride = page * width
        p.key_scales, p.value_scales, p.scale_block_stride = s["k_scales"].data_ptr(), s["v_scales"].data_ptr(), case["kv_heads"]
    if page:
        p.block_table, p.block_tokens, p.block_table_stride = s["table"].data_ptr(), page, s["table"].shape[1]
        p.pool_blocks = s["k"].shape[0]
    p.kv_tokens, p.kv_tokens_max, p.query_start_from_end = s["kv_tokens"].data_ptr(), max(s["lengths"]), 1
    if case["bias"]:
        p.slopes = s["slopes"].data_ptr()
    if case["mask"] != "none":
        p.row_first, p.row_end = s["first"].data_ptr(), s["end"].data_ptr()
    lib.yvx_cuda_scored_plan(C.byref(p), torch.cuda.get_device_properties(DEV).multi_processor_count)
    s["work"] = torch.empty(max(16, lib.yvx_cuda_scored_workspace_bytes(C.byref(p))), dtype=torch.uint8, device=DEV)
    p.workspace, p.workspace_bytes, p.status = s["work"].data_ptr(), s["work"].numel(), s["status"].data_ptr()
    s["args"] = p


def _call(s):
    stream = torch.cuda.current_stream().cuda_stream
    kind, lib, args = s["case"]["kind"], s["lib"], C.byref(s["args"])
    if kind == "append8":
        rc, out = lib.yvx_cuda_kv8_append(args, stream), [s["k_codes"], s["k_scales"], s["v_codes"], s["v_scales"]]
    elif kind == "pages":
        rc, out = lib.yvx_cuda_kv_pages_copy(args, stream, None), s["pools"]
    else:
        rc, out = lib.yvx_cuda_scored_attention(args, stream, None), s["out"]
    if rc:
        raise RuntimeError(lib.yvx_cuda_last_error_text().decode())
    return out


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        _handle(s)
    return s


def run(state):
    if own:
        return _call(state)
    return {"append8": _plain_append, "attend": _plain_attend, "pages": _plain_pages}[state["case"]["kind"]](state)


# ---- the definition in 64 bits --------------------------------------------------------------------


def _round_code(x, cache):
    """Nearest code value, ties to even: whole numbers, or e4m3's grid (3 fraction bits, smallest exponent -6)."""
    if cache == "i8":
        return torch.round(x)
    _, e = torch.frexp(x.abs())
    step = torch.exp2((e - 1).clamp(min=-6).double() - 3)
    return torch.round(x / step) * step


def _exact_append(s):
    case, out = s["case"], []
    page, limit = case["page"], LIMIT[case["cache"]]
    for x in ("k", "v"):
        codes, scales = s[x + "_codes"].double(), s[x + "_scales"].double()
        for b, n in enumerate(s["before"]):
            for j in range(n // page, -(-(n + case["rows"]) // page)):
                block = int(s["table"][b, j])
                lo, hi = max(n, j * page), min(n + case["rows"], (j + 1) * page)
                new = s[x][b, lo - n:hi - n].double()                       # [slot][head][dim]
                a, e = torch.frexp(new.abs().amax((0, 2)) / limit)          # [head]: a in [1/2, 1)
                e = torch.where(a == 0.5, e - 1, e).clamp(min=-126)
                fresh = torch.exp2(torch.where(a == 0, torch.full_like(e, -126), e).double())
                kept = lo - j * page
                if kept:
                    fresh = torch.maximum(fresh, scales[block])
                    codes[block, :, :kept] = _round_code(codes[block, :, :kept] * (scales[block] / fresh)[:, None, None], case["cache"])
                codes[block, :, kept:hi - j * page] = _round_code(new.permute(1, 0, 2) / fresh[:, None, None], case["cache"])
                scales[block] = fresh
        out += [codes if case["cache"] == "e4m3" else codes.to(torch.int8), scales]
    return out


def _exact_attend(s):
    case = s["case"]
    first, end, position = (torch.from_numpy(np.ascontiguousarray(x)).to(DEV) for x in _ranges(case))
    group = case["heads"] // case["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    for b, n in enumerate(s["lengths"]):
        lo, hi = int(first[b].min()), int(end[b].max())
        if hi <= lo:
            continue
        keys, values = (_session_rows(s, x, b, torch.float64)[:, lo:hi] for x in ("k", "v"))
        token = torch.arange(lo, hi, device=DEV)
        for at in range(0, case["rows"], 2048):
            cut = slice(at, min(case["rows"], at + 2048))
            hidden = (token[None] < first[b, cut, None]) | (token[None] >= end[b, cut, None])
            for h in range(case["heads"]):
                logit = torch.einsum("rd,td->rt", s["q"][b, cut, h].double(), keys[h // group]) * case["dim"] ** -0.5
                if case["cap"]:
                    e = torch.exp(-2 * logit.abs() / case["cap"])
                    logit = torch.sign(logit) * case["cap"] * (1 - e) / (1 + e)
                if case["bias"]:
                    logit -= s["slopes"][h].double() * (position[b, cut, None] - token[None]).abs()
                logit[hidden] = -math.inf
                norm = torch.logsumexp(logit, -1, keepdim=True)
                p = torch.exp(logit - torch.where(norm == -math.inf, torch.zeros_like(norm), norm))
                out[b, cut, h] = p @ values[h // group]
    return out


def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "pages":
        out = [pool.clone() for pool in s["pools"]]
        for was, pool in zip(s["pools"], out):
            for a, b, r in s["moves"]:
                pool[b, :r] = was[a, :r]
        return out
    return _exact_append(s) if case["kind"] == "append8" else _exact_attend(s)
