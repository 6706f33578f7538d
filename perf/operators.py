"""The long-context operators as cases that can be timed and checked.

A case names a family, its sizes and its storage type.  `prepare` makes what a serving
engine holds before the call (activations, the paged KV cache, its block tables), `run`
makes one pass, in plain torch or, where `own` is set, through `nano_vllm_cpp_amd.ops`,
and `exact` computes the same outputs in 64 bits.

Families:
  window   paged attention over a sliding window and a few first keys (sinks)
  prefix   paged attention of a decode batch whose sequences share long prefixes
  fork     sequences forked with their pages shared (the last, partial page copied), then freed
  copy     pages of a cache copied to others, in all layers
  compact  a cache's used pages moved together, block tables and reference counts with them
  rotary   rotary positions (half or interleaved pairs, part of the head, far positions), KV store
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HEADS = {"14/2/64": (14, 2, 64), "28/4/128": (28, 4, 128), "32/8/128": (32, 8, 128)}  # q heads, kv heads, head size
SMALL, WIDE, MANY = sorted(HEADS)
EPS = 1e-6


def listed() -> list[dict]:
    return [
        # interactive generation on a small model: one token, latency
        dict(name="window_decode_1", family="window", ctx="16384", new="1", window=2048, sinks=4, heads=SMALL,
             page=256, dtype="f16"),
        # a serving engine's decode step over long ragged contexts, some rows of the batch padding
        dict(name="window_decode_256", family="window", ctx="ragged:256:16384", new="1", window=4096, sinks=4,
             heads=WIDE, page=256, dtype="bf16"),
        # a packed prefill of ragged prompts
        dict(name="window_prefill", family="window", ctx="8192,3001,777", new="all", window=2048, sinks=4, heads=WIDE,
             page=256, dtype="f16"),
        # chunks of two prompts after cached keys, on the reference's own cache type
        dict(name="window_chunk_f32", family="window", ctx="5700,6100", new="700,300", window=2048, sinks=16,
             heads=MANY, page=32, dtype="f32"),
        # a few samples of one prompt on a small model: latency
        dict(name="prefix_8", family="prefix", sizes="8", prefix="1000", tail=64, heads=SMALL, page=16, dtype="f16"),
        # a decode batch under one long system prompt
        dict(name="prefix_256", family="prefix", sizes="256", prefix="8192", tail=1024, heads=WIDE, page=256,
             dtype="bf16"),
        # a decode batch of several prompts, sampled different numbers of times
        dict(name="prefix_groups", family="prefix", sizes="96,17,40,7", prefix="4096,1999,12288,300", tail=2048,
             heads=MANY, page=64, dtype="f16"),
        # a request asks for four more samples: all layers of a model
        dict(name="fork_4", family="fork", forks=4, caches=56, pages=64, heads=WIDE, page=256, dtype="f16"),
        # a pool half empty after a burst of requests
        dict(name="compact_768", family="compact", caches=16, pages=768, used=420, moves=180, heads=WIDE, page=256,
             dtype="f16"),
        # a decode step's positions far into their contexts, half of each head rotated, KV store
        dict(name="rotary_decode_256", family="rotary", tokens=256, far=1000000, rot=64, interleaved=True, scale=1.0,
             norm=False, store=True, heads=MANY, dtype="f16"),
        # a full prefill chunk, frequencies scaled for a longer context, KV store
        dict(name="rotary_prefill_16384", family="rotary", tokens=16384, far=131072, rot=128, interleaved=False,
             scale=1.1386, norm=False, store=True, heads=WIDE, dtype="bf16"),
        # an odd number of prompt tokens, per-head norm first, no store
        dict(name="rotary_norm_f32", family="rotary", tokens=1021, far=40000, rot=32, interleaved=False, scale=1.0,
             norm=True, store=False, heads=SMALL, dtype="f32"),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    family = rng.choice(["window", "window", "window", "prefix", "prefix", "fork", "copy", "compact", "rotary"])
    heads, dtype = rng.choice(sorted(HEADS)), rng.choice(["f32", "f16", "bf16"])
    page = rng.choice([16, 32, 64, 256])
    if family == "window":
        c = dict(family=family, window=_log_int(rng, 16, 4096), sinks=rng.choice([0, 1, 4, 64, 100]), heads=heads,
                 page=page, dtype=dtype)
        kind = rng.choice(["one", "batch", "prefill", "chunk"])
        if kind == "one":
            return dict(c, ctx=str(_log_int(rng, 1, 32768)), new="1")
        if kind == "batch":
            return dict(c, ctx="ragged:%d:%d" % (_log_int(rng, 2, 200), _log_int(rng, 64, 16384)), new="1")
        lens = [_log_int(rng, 40, 3000) for _ in range(rng.randint(1, 3))]
        if kind == "prefill":
            return dict(c, ctx=",".join(map(str, lens)), new="all")
        return dict(c, ctx=",".join(map(str, lens)), new=",".join(str(_log_int(rng, 1, min(n, 500))) for n in lens))
    if family == "prefix":
        groups = rng.randint(1, 4)
        sizes = [_log_int(rng, 1, 50 if groups > 1 else 200) for _ in range(groups)]
        return dict(family=family, sizes=",".join(map(str, sizes)),
                    prefix=",".join(str(_log_int(rng, 30, 6000)) for _ in sizes), tail=_log_int(rng, 1, 1000),
                    heads=heads, page=page, dtype=dtype)
    if family in ("fork", "copy"):
        pages = _log_int(rng, 40, 150)
        return dict(family=family, forks=_log_int(rng, 1, 24), caches=2 * rng.randint(1, 28), pages=pages, heads=heads,
                    page=page, dtype=dtype)
    if family == "compact":
        caches, pages = 2 * rng.randint(1, 8), _log_int(rng, 30, 700)
        used = rng.randint(pages // 4, 3 * pages // 4)
        most = int(1.5e9 / (caches * page * 4096))  # at up to 4096 bytes a key: what the listed case moves
        return dict(family=family, caches=caches, pages=pages, used=used,
                    moves=rng.randint(1, max(1, min(used, pages - used, most))), heads=heads, page=page, dtype=dtype)
    hd = HEADS[heads][2]
    return dict(family=family, tokens=_log_int(rng, 1, 12000), far=_log_int(rng, 1000, 1000000),
                rot=rng.choice([hd, hd // 2]), interleaved=rng.random() < 0.5, scale=rng.choice([1.0, 1.2]),
                norm=rng.random() < 0.4, store=rng.random() < 0.6, heads=heads, dtype=dtype)


# ---------------------------------------------------------------------------
# sizes that follow from a case
# ---------------------------------------------------------------------------
def _ints(text: str) -> list[int]:
    return [int(v) for v in text.split(",")]


def _batch(case: dict) -> tuple[np.ndarray, np.ndarray]:
    """(keys, new tokens) of each sequence of a window case: part of its shape, not of its inputs."""
    if case["ctx"].startswith("ragged"):
        _, n, most = case["ctx"].split(":")
        ctx = np.random.default_rng(int(n)).integers(1, int(most) + 1, int(n))
        ctx[::32][1:] = 0  # padding rows of the batch
        return ctx, np.ones(int(n), np.int64)
    ctx = np.array(_ints(case["ctx"]))
    return ctx, ctx.copy() if case["new"] == "all" else np.array(_ints(case["new"]))


def _groups(case: dict):
    """(group sizes, prefix lengths, each sequence's key count) of a prefix case."""
    sizes, prefix = np.array(_ints(case["sizes"])), np.array(_ints(case["prefix"]))
    tail = np.random.default_rng(int(sizes.sum())).integers(1, case["tail"] + 1, int(sizes.sum()))
    return sizes, prefix, np.repeat(prefix, sizes) + tail


def _visible(n: np.ndarray, window: int, sinks: int) -> np.ndarray:
    """How many keys a token with n keys sees."""
    return np.minimum(n, window) + np.minimum(np.maximum(n - window, 0), sinks)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _normal(g, shape, dtype, mean: float = 0.0, std: float = 1.0) -> torch.Tensor:
    out = torch.empty(shape, dtype=dtype, device=DEV)
    flat = out.view(-1)
    for i in range(0, flat.numel(), 1 << 28):  # in pieces: no fp32 copy of a whole cache
        part = flat[i:i + (1 << 28)]
        part.copy_(torch.randn(part.numel(), generator=g, device=DEV).mul_(std).add_(mean))
    return out


def _dev(a, dtype=torch.int32) -> torch.Tensor:
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV, dtype)


def _prepare_window(case: dict, g, r) -> dict:
    qh, kvh, hd = HEADS[case["heads"]]
    page, dt = case["page"], TYPES[case["dtype"]]
    ctx, new = _batch(case)
    table = np.full((len(ctx), max(1, -(-int(ctx.max()) // page))), -1, np.int32)
    seen = np.zeros_like(table, dtype=bool)  # pages that a token of the batch sees; the others are freed
    for s, (n, k) in enumerate(zip(ctx, new)):
        first = max(0, n - k + 1 - case["window"])
        for j in range(-(-int(n) // page)):
            seen[s, j] = j * page < case["sinks"] or (j + 1) * page > first
    used = int(seen.sum())
    table[seen] = r.permutation(used).astype(np.int32)
    seq = np.repeat(np.arange(len(ctx)), new)
    key_len = np.concatenate([np.arange(n - k, n) + 1 for n, k in zip(ctx, new)])
    key_len[np.repeat(ctx == 0, new)] = 0
    return dict(case=case, q=_normal(g, (int(new.sum()), qh, hd), dt), k_cache=_normal(g, (used * page, kvh, hd), dt),
                v_cache=_normal(g, (used * page, kvh, hd), dt), query_seq=_dev(seq), key_len=_dev(key_len),
                table=_dev(table), cu=np.concatenate([[0], np.cumsum(new)]).astype(np.int32),
                decode=bool((new == 1).all()))


def _prepare_prefix(case: dict, g, r) -> dict:
    qh, kvh, hd = HEADS[case["heads"]]
    page, dt = case["page"], TYPES[case["dtype"]]
    sizes, prefix, key_len = _groups(case)
    table = np.full((len(key_len), -(-int(key_len.max()) // page)), -1, np.int32)
    group = np.repeat(np.arange(len(sizes)), sizes)
    start = np.concatenate([[0], np.cumsum(sizes)])
    # the prefix's full pages are one set for the group; the page that it ends in is each sequence's
    # own (keys are appended to it), with the same prefix keys in it
    shared = prefix // page
    need = -(-key_len // page) - shared[group]
    pages = r.permutation(int(shared.sum() + need.sum())).astype(np.int32)
    at = int(shared.sum())
    firsts = np.concatenate([[0], np.cumsum(shared)])
    for s, n in enumerate(key_len):
        p = group[s]
        table[s, :shared[p]] = pages[firsts[p]:firsts[p + 1]]
        table[s, shared[p]:shared[p] + need[s]] = pages[at:at + need[s]]
        at += need[s]
    k_cache = _normal(g, (len(pages) * page, kvh, hd), dt)
    v_cache = _normal(g, (len(pages) * page, kvh, hd), dt)
    for p, n in enumerate(prefix % page):
        if n:  # as forks leave it: the first sequence's rows in every other one's page
            own_pages = _dev(table[start[p]:start[p + 1], shared[p]], torch.int64)
            for c in (k_cache, v_cache):
                c = c.view(-1, page, kvh, hd)
                c[own_pages, :int(n)] = c[own_pages[:1], :int(n)].clone()
    return dict(case=case, q=_normal(g, (len(key_len), qh, hd), dt), k_cache=k_cache, v_cache=v_cache,
                query_seq=_dev(np.arange(len(key_len))), key_len=_dev(key_len), table=_dev(table),
                prefix=prefix.astype(np.int32), start=start.astype(np.int32))


def _caches(g, case: dict) -> torch.Tensor:
    _, kvh, hd = HEADS[case["heads"]]
    return _normal(g, (case["caches"], case["pages"] * case["page"], kvh, hd), TYPES[case["dtype"]])


def _fork_lens(case: dict) -> tuple[int, np.ndarray]:
    """(parents, their key counts): forks take them in turn."""
    parents = max(1, min(case["forks"], 5))
    most = (case["pages"] - case["forks"]) // parents * case["page"]
    return parents, np.random.default_rng(case["forks"] + case["pages"]).integers(1, most, parents)


def _prepare_pages(case: dict, g, r) -> dict:
    stack, pages, page = _caches(g, case), case["pages"], case["page"]
    s = dict(case=case, stack=stack, caches=list(stack.unbind(0)))
    if case["family"] == "copy":
        p = r.permutation(pages).astype(np.int32)
        n = min(case["forks"], pages // 2)
        return dict(s, src=p[:n].copy(), dst=p[n:2 * n].copy())
    if case["family"] == "fork":
        parents, lens = _fork_lens(case)
        n, most = case["forks"], -(-int(lens.max()) // page) + 4
        rows = r.permutation(parents + n).astype(np.int32)
        table, ref, key_len = np.full((parents + n, most), -1, np.int32), np.zeros(pages, np.int32), np.zeros(parents + n)
        p = r.permutation(pages).astype(np.int32)
        at = 0
        for i, k in enumerate(lens):
            used = -(-int(k) // page)
            table[rows[i], :used] = p[at:at + used]
            ref[p[at:at + used]] = 1
            key_len[rows[i]] = k
            at += used
        return dict(s, table=_dev(table), ref=_dev(ref), key_len=_dev(key_len), child=rows[parents:].copy(),
                    parent=rows[np.arange(n) % parents].copy())
    used, moves = case["used"], case["moves"]
    holes = r.permutation(used)[:moves]  # free pages below the number of used ones
    high = used + r.permutation(pages - used)[:moves]
    ref = np.zeros(pages, np.int32)
    ref[:used] = 1
    ref[holes] = 0
    ref[high] = 1
    live = r.permutation(np.flatnonzero(ref)).astype(np.int32)
    ref[live[::7]] = 2  # pages that two sequences share
    entries = np.concatenate([live, live[::7]])
    cols = 16
    table = np.full((-(-len(entries) // 11), cols), -1, np.int32)  # 11 pages a sequence, the last one fewer
    for i in range(len(table)):
        row = entries[i * 11:(i + 1) * 11]
        table[i, :len(row)] = row
    return dict(s, table=_dev(table), ref=_dev(ref), table_out=_dev(table), ref_out=_dev(ref))


def _prepare_rotary(case: dict, g, r) -> dict:
    qh, kvh, hd = HEADS[case["heads"]]
    t, dt = case["tokens"], TYPES[case["dtype"]]
    qkv = _normal(g, (t, (qh + 2 * kvh) * hd), dt)
    i = torch.arange(case["rot"] // 2, dtype=torch.float64, device=DEV)
    s = dict(case=case, qkv=qkv, positions=torch.randint(0, case["far"], (t,), generator=g, device=DEV),
             inv_freq=1e6 ** (-2.0 * i / case["rot"]), q_out=torch.empty((t, qh * hd), dtype=dt, device=DEV),
             q_w=_normal(g, (hd,), dt, 1.0, 0.1) if case["norm"] else None,
             k_w=_normal(g, (hd,), dt, 1.0, 0.1) if case["norm"] else None)
    if not case["store"]:
        return dict(s, k_out=torch.empty((t, kvh * hd), dtype=dt, device=DEV))
    slots = r.permutation(t + 64)[:t].astype(np.int32)
    slots[3::50] = -1  # tokens that are not stored
    return dict(s, slots=_dev(slots), k_cache=_normal(g, (t + 64, kvh, hd), dt),
                v_cache=_normal(g, (t + 64, kvh, hd), dt))


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    r = np.random.default_rng(seed)
    make = dict(window=_prepare_window, prefix=_prepare_prefix, rotary=_prepare_rotary)
    return make.get(case["family"], _prepare_pages)(case, g, r)


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _softmax_product(scores: torch.Tensor, seen: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
    """softmax over the seen keys (last dim), times v; zeros where none is seen."""
    scores = torch.where(seen, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    return (p @ v) / p.sum(-1, keepdim=True).clamp_min(1e-30)


def _attend_gathered(s: dict, keys: torch.Tensor, seen: torch.Tensor) -> torch.Tensor:
    """Each token over its own list of keys [tokens, n], those of them that are seen."""
    q, page = s["q"], s["case"]["page"]
    t, qh, hd = q.shape
    kvh = s["k_cache"].shape[1]
    entry = s["table"][s["query_seq"].long()[:, None], keys // page]
    rows = torch.where(seen, entry.long() * page + keys % page, torch.zeros_like(keys))
    k = s["k_cache"][rows].float().permute(0, 2, 3, 1).contiguous()  # [t, kvh, hd, n]
    v = s["v_cache"][rows].float().permute(0, 2, 1, 3).contiguous()
    scores = (q.float().view(t, kvh, qh // kvh, hd) @ k) * hd ** -0.5
    return _softmax_product(scores, seen[:, None, None, :], v).reshape(t, qh, hd).to(q.dtype)


def _attend_packed(s: dict) -> torch.Tensor:
    """Every token against the packed keys of all sequences, the others' and unseen ones masked."""
    c, q = s["case"], s["q"]
    t, qh, hd = q.shape
    kvh, g = s["k_cache"].shape[1], qh // s["k_cache"].shape[1]
    entries = s["table"].reshape(-1).long()
    live = (entries >= 0).nonzero().view(-1)
    at = (live[:, None] * c["page"] + torch.arange(c["page"], device=DEV)).view(-1)  # (sequence, key) as one number
    width = s["table"].shape[1] * c["page"]
    seq, key = at // width, at % width
    rows = entries[at // c["page"]] * c["page"] + at % c["page"]
    k = s["k_cache"][rows].float().permute(1, 2, 0).contiguous()  # [kvh, hd, n]
    v = s["v_cache"][rows].float().permute(1, 0, 2).contiguous()
    scores = (q.float().view(t, kvh, g, hd).permute(1, 2, 0, 3).reshape(kvh, g * t, hd) @ k) * hd ** -0.5
    n = s["key_len"].long()[:, None]
    seen = (s["query_seq"].long()[:, None] == seq) & (key < n) & ((key < c["sinks"]) | (key >= n - c["window"]))
    out = _softmax_product(scores, seen.repeat(g, 1), v)
    return out.view(kvh, g, t, hd).permute(2, 0, 1, 3).reshape(t, qh, hd).to(q.dtype)


def _plain_window(s: dict) -> torch.Tensor:
    if not s["decode"]:
        return _attend_packed(s)
    c, n = s["case"], s["key_len"].long()[:, None]
    most = s["table"].shape[1] * c["page"]
    window, sinks = min(c["window"], most), min(c["sinks"], most)
    first = torch.arange(sinks, device=DEV).expand(n.shape[0], -1)
    last = n - window + torch.arange(window, device=DEV)
    keys = torch.cat([first, last.clamp_min(0)], 1)
    return _attend_gathered(s, keys, torch.cat([first < (n - window), last >= 0], 1))


def _plain_prefix(s: dict) -> torch.Tensor:
    n = s["key_len"].long()[:, None]
    keys = torch.arange(s["table"].shape[1] * s["case"]["page"], device=DEV).expand(n.shape[0], -1)
    return _attend_gathered(s, keys, keys < n)


def _plain_copy(s: dict):
    pages = s["stack"].view(s["case"]["caches"], s["case"]["pages"], -1)
    pages[:, _dev(s["dst"], torch.int64)] = pages[:, _dev(s["src"], torch.int64)]
    return s["stack"]


def _plain_fork(s: dict):
    c, table, ref, key_len = s["case"], s["table"], s["ref"], s["key_len"]
    parent, child = _dev(s["parent"], torch.int64), _dev(s["child"], torch.int64)
    n = key_len[parent].long()
    full, rest = n // c["page"], n % c["page"]
    column = torch.arange(table.shape[1], device=DEV)
    old = table[parent].long()
    shared = column < full[:, None]
    free = (ref == 0).nonzero().view(-1)
    new = torch.where(rest > 0, free[(torch.cumsum(rest > 0, 0) - 1).clamp_min(0)], -1)
    table[child] = torch.where(shared, old, torch.where((column == full[:, None]) & (rest > 0)[:, None], new[:, None],
                                                        -1)).int()
    key_len[child] = n.int()
    ref.index_add_(0, old[shared], torch.ones_like(old[shared], dtype=torch.int32))
    ref[new[rest > 0]] = 1
    # the last page's rows, of every cache
    rows = torch.arange(c["page"], device=DEV)
    take = rows < rest[:, None]
    last = old.gather(1, full.clamp_max(table.shape[1] - 1)[:, None])
    src, dst = (last * c["page"] + rows)[take], (new[:, None] * c["page"] + rows)[take]
    s["stack"][:, dst] = s["stack"][:, src]
    # the children end: their pages are given back
    gone = table[child].long()
    ref.index_add_(0, gone[gone >= 0], torch.full_like(gone[gone >= 0], -1, dtype=torch.int32))
    table[child], key_len[child] = -1, 0
    return new.int(), table, ref, key_len, s["stack"]


def _plain_compact(s: dict):
    ref, table = s["ref"], s["table"].long()
    used = int((ref > 0).sum())
    src = used + (ref[used:] > 0).nonzero().view(-1)
    dst = (ref[:used] == 0).nonzero().view(-1)
    where = torch.arange(len(ref), device=DEV)
    where[src] = dst
    pages = s["stack"].view(s["case"]["caches"], s["case"]["pages"], -1)
    pages[:, dst] = pages[:, src]
    table_out = torch.where(table >= 0, where[table.clamp_min(0)], -1).int()
    ref_out = ref.clone()
    ref_out[dst] = ref[src]
    ref_out[src] = 0
    return table_out, ref_out, s["stack"]


def _plain_rotary(s: dict):
    c = s["case"]
    qh, kvh, hd = HEADS[c["heads"]]
    t, r = c["tokens"], c["rot"]
    angle = s["positions"].double()[:, None] * s["inv_freq"]
    cos, sin = (torch.cos(angle) * c["scale"]).float()[:, None], (torch.sin(angle) * c["scale"]).float()[:, None]
    x = s["qkv"][:, :(qh + kvh) * hd].float().view(t, qh + kvh, hd)
    if c["norm"]:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        x = torch.cat([x[:, :qh] * s["q_w"].float(), x[:, qh:] * s["k_w"].float()], 1)
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if c["interleaved"] else (x[..., :r // 2], x[..., r // 2:r])
    y = [a * cos - b * sin, b * cos + a * sin]
    y = torch.stack(y, -1).flatten(-2) if c["interleaved"] else torch.cat(y, -1)
    y = torch.cat([y, x[..., r:]], -1).to(s["qkv"].dtype)
    q, k = y[:, :qh].reshape(t, -1), y[:, qh:].reshape(t, -1)
    if not c["store"]:
        return q, k
    kept = s["slots"] >= 0
    at = s["slots"][kept].long()
    s["k_cache"][at] = k[kept].view(-1, kvh, hd)
    s["v_cache"][at] = s["qkv"][:, (qh + kvh) * hd:][kept].view(-1, kvh, hd)
    return q, s["k_cache"], s["v_cache"]


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------
def _own_rotary(ops, s: dict):
    c = s["case"]
    qh, kvh, hd = HEADS[c["heads"]]
    q, k, v = s["qkv"][:, :qh * hd], s["qkv"][:, qh * hd:(qh + kvh) * hd], s["qkv"][:, (qh + kvh) * hd:]
    if c["store"]:
        ops.rotary_store_kv(q, k, v, s["positions"], s["inv_freq"], qh, kvh, hd, s["k_cache"], s["v_cache"], s["slots"],
                            interleaved=c["interleaved"], attn_scale=c["scale"], q_w=s["q_w"], k_w=s["k_w"], eps=EPS,
                            q_out=s["q_out"])
        return s["q_out"], s["k_cache"], s["v_cache"]
    ops.rotary(q, k, s["positions"], s["inv_freq"], qh, kvh, hd, interleaved=c["interleaved"], attn_scale=c["scale"],
               q_w=s["q_w"], k_w=s["k_w"], eps=EPS, q_out=s["q_out"], k_out=s["k_out"])
    return s["q_out"], s["k_out"]


def _run_own(s: dict):
    from nano_vllm_cpp_amd import ops

    c = s["case"]
    if c["family"] == "rotary":
        return _own_rotary(ops, s)
    if c["family"] == "window":
        return ops.window_attention(s["q"], s["k_cache"], s["v_cache"], s["query_seq"], s["key_len"], s["table"],
                                    c["page"], s["q"].shape[2] ** -0.5, c["window"], c["sinks"],
                                    max_query_len=1 if s["decode"] else 0, cu_seqlens=None if s["decode"] else s["cu"])
    if c["family"] == "prefix":
        return ops.prefix_attention(s["q"], s["k_cache"], s["v_cache"], s["query_seq"], s["key_len"], s["table"],
                                    c["page"], s["q"].shape[2] ** -0.5, s["prefix"], s["start"])
    if c["family"] == "copy":
        ops.copy_pages(s["caches"], s["src"], s["dst"], c["page"])
        return s["stack"]
    if c["family"] == "fork":
        new = ops.fork_pages(s["caches"], s["table"], s["key_len"], s["ref"], s["parent"], s["child"], c["page"])
        ops.free_pages(s["table"], s["key_len"], s["ref"], s["child"], c["page"])
        return new, s["table"], s["ref"], s["key_len"], s["stack"]
    ops.compact_pages(s["caches"], s["table"], s["ref"], c["page"], table_out=s["table_out"], ref_out=s["ref_out"])
    return s["table_out"], s["ref_out"], s["stack"]


def run(state: dict):
    if own:
        return _run_own(state)
    return dict(window=_plain_window, prefix=_plain_prefix, copy=_plain_copy, fork=_plain_fork, compact=_plain_compact,
                rotary=_plain_rotary)[state["case"]["family"]](state)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case: dict) -> dict:
    qh, kvh, hd = HEADS[case["heads"]]
    e, row = (4 if case["dtype"] == "f32" else 2), kvh * hd
    family = case["family"]
    if family == "window":
        ctx, new = _batch(case)
        tokens = int(new[ctx > 0].sum())
        pairs = sum(int(_visible(np.arange(n - k, n) + 1, case["window"], case["sinks"]).sum())
                    for n, k in zip(ctx, new) if n > 0)
        span = np.minimum(ctx, case["window"] + new - 1)  # the keys that some token of the sequence sees
        keys = int((span + np.minimum(np.maximum(ctx - span, 0), case["sinks"])).sum())
        return dict(bytes=2 * keys * row * e + (tokens + len(ctx)) * qh * hd * e, flops=4.0 * pairs * qh * hd)
    if family == "prefix":
        sizes, prefix, n = _groups(case)
        keys = int(prefix.sum() + (n - np.repeat(prefix, sizes)).sum())
        return dict(bytes=2 * keys * row * e + 2 * len(n) * qh * hd * e, flops=4.0 * int(n.sum()) * qh * hd)
    if family == "rotary":
        t = case["tokens"]
        return dict(bytes=t * (2 * qh * hd + (4 if case["store"] else 2) * row) * e, flops=6.0 * t * (qh + kvh) * hd)
    page = case["page"] * row * e
    if family == "copy":
        return dict(bytes=2 * min(case["forks"], case["pages"] // 2) * page * case["caches"], flops=0)
    if family == "fork":
        parents, lens = _fork_lens(case)
        rest = int((lens[np.arange(case["forks"]) % parents] % case["page"]).sum())
        return dict(bytes=2 * rest * row * e * case["caches"] + 4 * case["pages"], flops=0)
    return dict(bytes=2 * case["moves"] * page * case["caches"] + 16 * case["pages"], flops=0)


# ---------------------------------------------------------------------------
# the outputs from their definitions, in 64 bits
# ---------------------------------------------------------------------------
def _exact_rows(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, seen: torch.Tensor) -> torch.Tensor:
    """q [t, qh, hd] over keys k, v [n, kvh, hd], of which token t sees seen[t]."""
    qh, hd = q.shape[1:]
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    for h in range(qh):
        kh = h // (qh // k.shape[1])
        w = q[:, h].double() @ k[:, kh].double().T.contiguous() / math.sqrt(hd)
        w.masked_fill_(~seen, -math.inf)
        some = seen.any(1)
        out[some, h] = torch.softmax(w[some], 1) @ v[:, kh].double()
    return out


def _exact_attention(s: dict, window: int, sinks: int) -> torch.Tensor:
    seq, key_len, table = (s[n].cpu().numpy() for n in ("query_seq", "key_len", "table"))
    page = s["case"]["page"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    for b in np.unique(seq):
        tokens = np.flatnonzero(seq == b)
        most = int(key_len[tokens].max())
        j = np.arange(most)
        j = j[table[b, j // page] >= 0]
        if not len(j):
            continue
        rows = torch.from_numpy(table[b, j // page].astype(np.int64) * page + j % page).to(DEV)
        n = key_len[tokens][:, None]
        seen = torch.from_numpy((j < n) & ((j < sinks) | (j >= n - window))).to(DEV)
        at = torch.from_numpy(tokens).to(DEV)
        out[at] = _exact_rows(s["q"][at], s["k_cache"][rows], s["v_cache"][rows], seen)
    return out


def _exact_rotary(s: dict):
    c = s["case"]
    qh, kvh, hd = HEADS[c["heads"]]
    t, r = c["tokens"], c["rot"]
    x = s["qkv"].double().view(t, qh + 2 * kvh, hd)
    heads = x[:, :qh + kvh].clone()
    if c["norm"]:
        heads /= torch.sqrt(heads.pow(2).sum(-1, keepdim=True) / hd + EPS)
        heads[:, :qh] *= s["q_w"].double()
        heads[:, qh:] *= s["k_w"].double()
    y = heads.clone()
    for i in range(r // 2):
        a, b = (2 * i, 2 * i + 1) if c["interleaved"] else (i, i + r // 2)
        z = torch.complex(heads[..., a], heads[..., b])
        angle = s["positions"].double() * s["inv_freq"][i]
        z = z * torch.polar(torch.full_like(angle, c["scale"]), angle)[:, None]
        y[..., a], y[..., b] = z.real, z.imag
    q, k = y[:, :qh].reshape(t, -1), y[:, qh:]
    if not c["store"]:
        return q, k.reshape(t, -1)
    k_cache, v_cache = s["k_cache"].double(), s["v_cache"].double()
    for i, slot in enumerate(s["slots"].tolist()):
        if slot >= 0:
            k_cache[slot], v_cache[slot] = k[i], x[i, qh + kvh:]
    return q, k_cache, v_cache


def exact(case: dict, seed: int):
    family = case["family"]
    if family not in ("window", "prefix", "rotary"):
        return None  # copies and whole numbers
    s = prepare(case, seed)
    if family == "rotary":
        return _exact_rotary(s)
    return _exact_attention(s, case["window"], case["sinks"]) if family == "window" else _exact_attention(s, 1 << 30, 0)
