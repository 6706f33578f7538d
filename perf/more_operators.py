"""The 4-bit KV cache's operators and the packed prompt's attention, as cases that can be timed and checked.

A case names a family, its sizes and its storage type.  `prepare` makes what a serving
engine holds before the call (activations, the paged 4-bit cache, its block tables), `run`
makes one pass, in plain torch or, where `own` is set, through `nano_vllm_cpp_amd.ops`,
and `exact` computes the same outputs in 64 bits.

Families:
  kv4     paged attention over a cache held in 4 bits: single tokens, a few tokens, chunks of prompts
  store   per-head norm, rotary positions and K and V appended to a 4-bit cache; the cache read back
  prompt  causal attention of packed prompts over their own K and V rows

A row of a 4-bit cache is one token: for each kv head head_dim / 2 bytes of codes (dimension 2 b in the low
half of byte b, 2 b + 1 in the high one), then for each kv head one 16-bit word for each 32 dimensions, then
zeros to a multiple of 16 bytes.  A word's upper 12 bits are those of an fp16 scale d, the lower four a
zero point z, and a code n stands for d (n - z), which fp16 holds exactly.
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
GROUP = 32  # dimensions of a scale
MOST_SCALE, LEAST_NORMAL = 4352.0, 2.0 ** -14


def listed() -> list[dict]:
    return [
        # interactive generation on a small model: one token, latency
        dict(name="kv4_decode_1", family="kv4", ctx="16384", new="1", heads=SMALL, page=256, dtype="f16"),
        # a serving engine's decode step over ragged contexts, some rows of the batch padding
        dict(name="kv4_decode_256", family="kv4", ctx="ragged:256:8192", new="1", heads=WIDE, page=256, dtype="bf16"),
        # the same in fp32, the reference's own activation type, on a small model with small pages
        dict(name="kv4_decode_48_f32", family="kv4", ctx="ragged:48:4096", new="1", heads=SMALL, page=16, dtype="f32"),
        # drafted tokens checked: five tokens of each sequence
        dict(name="kv4_verify_32", family="kv4", ctx="ragged:32:4096", new="5", heads=MANY, page=64, dtype="bf16"),
        # chunks of two prompts over what the cache holds of them
        dict(name="kv4_chunk", family="kv4", ctx="8192,4001", new="1000,700", heads=WIDE, page=256, dtype="f16"),
        # a decode batch's new tokens, interleaved pairs
        dict(name="store_decode_256", family="store", tokens=256, far=100000, rot=64, interleaved=True, scale=1.0,
             norm=False, heads=MANY, dtype="f16"),
        # a full prefill chunk, frequencies scaled for a longer context
        dict(name="store_prefill_16384", family="store", tokens=16384, far=131072, rot=128, interleaved=False,
             scale=1.1386, norm=False, heads=WIDE, dtype="bf16"),
        # an odd number of prompt tokens, per-head norm first
        dict(name="store_norm_f32", family="store", tokens=1021, far=40000, rot=32, interleaved=False, scale=1.0,
             norm=True, heads=SMALL, dtype="f32"),
        # one short prompt on a small model: latency
        dict(name="prompt_37", family="prompt", lens="37", heads=SMALL, dtype="f16"),
        # a packed batch of ragged prompts, down to a single token
        dict(name="prompt_ragged", family="prompt", lens="4096,1500,777,64,1", heads=WIDE, dtype="bf16"),
        # one long prompt
        dict(name="prompt_8192", family="prompt", lens="8192", heads=MANY, dtype="f16"),
        # the reference's own activation type
        dict(name="prompt_f32", family="prompt", lens="1000,300,129", heads=MANY, dtype="f32"),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    family = rng.choice(["kv4", "kv4", "kv4", "store", "prompt", "prompt"])
    heads, dtype = rng.choice(sorted(HEADS)), rng.choice(["f32", "f16", "bf16"])
    if family == "kv4":
        c = dict(family=family, heads=heads, page=rng.choice([16, 32, 64, 256]), dtype=dtype)
        kind = rng.choice(["one", "batch", "few", "chunk"])
        if kind == "one":
            return dict(c, ctx=str(_log_int(rng, 1, 32768)), new="1")
        if kind == "batch":
            return dict(c, ctx="ragged:%d:%d" % (_log_int(rng, 2, 128), _log_int(rng, 64, 8000)), new="1")
        if kind == "few":
            return dict(c, ctx="ragged:%d:%d" % (_log_int(rng, 1, 24), _log_int(rng, 64, 4000)), new=str(rng.randint(2, 8)))
        lens = [_log_int(rng, 40, 6000) for _ in range(rng.randint(1, 3))]
        return dict(c, ctx=",".join(map(str, lens)), new=",".join(str(_log_int(rng, 1, min(n, 700))) for n in lens))
    if family == "store":
        hd = HEADS[heads][2]
        return dict(family=family, tokens=_log_int(rng, 1, 12000), far=_log_int(rng, 1000, 1000000),
                    rot=rng.choice([hd, hd // 2]), interleaved=rng.random() < 0.5, scale=rng.choice([1.0, 1.2]),
                    norm=rng.random() < 0.4, heads=heads, dtype=dtype)
    prompts = rng.randint(1, 5)
    lens = [_log_int(rng, 1, 8000 // prompts) for _ in range(prompts)]
    return dict(family=family, lens=",".join(map(str, lens)), heads=heads, dtype=dtype)


# ---------------------------------------------------------------------------
# sizes that follow from a case
# ---------------------------------------------------------------------------
def _ints(text: str) -> list[int]:
    return [int(v) for v in text.split(",")]


def _row_bytes(kvh: int, hd: int) -> int:
    return -(-kvh * (hd // 2 + hd // GROUP * 2) // 16) * 16


def _batch(case: dict) -> tuple[np.ndarray, np.ndarray]:
    """(keys, new tokens) of each sequence of a kv4 case: part of its shape, not of its inputs."""
    if case["ctx"].startswith("ragged"):
        _, n, most = case["ctx"].split(":")
        new = int(case["new"])
        ctx = np.random.default_rng(int(n)).integers(new, int(most) + 1, int(n))
        ctx[::32][1:] = 0  # padding rows of the batch
        return ctx, np.full(int(n), new, np.int64)
    return np.array(_ints(case["ctx"])), np.array(_ints(case["new"]))


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _normal(g, shape, dtype, mean: float = 0.0, std: float = 1.0) -> torch.Tensor:
    return torch.randn(shape, generator=g, device=DEV).mul_(std).add_(mean).to(dtype)


def _dev(a, dtype=torch.int32) -> torch.Tensor:
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV, dtype)


def _cache(g, rows: int, kvh: int, hd: int) -> torch.Tensor:
    """A 4-bit cache of normal values."""
    out = torch.zeros((rows, _row_bytes(kvh, hd)), dtype=torch.uint8, device=DEV)
    for i in range(0, rows, 1 << 17):  # in pieces: no fp32 copy of a whole cache
        n = min(1 << 17, rows - i)
        out[i:i + n] = _pack(torch.randn((n, kvh, hd), generator=g, device=DEV))
    return out


def _prepare_kv4(case: dict, g, r) -> dict:
    qh, kvh, hd = HEADS[case["heads"]]
    page = case["page"]
    ctx, new = _batch(case)
    pages = -(-ctx // page)
    table = np.full((len(ctx), max(1, int(pages.max()))), -1, np.int32)
    held = np.arange(table.shape[1]) < pages[:, None]
    table[held] = r.permutation(int(pages.sum())).astype(np.int32)
    seq = np.repeat(np.arange(len(ctx)), new)
    key_len = np.concatenate([np.arange(n - k, n) + 1 for n, k in zip(ctx, new)])
    key_len[np.repeat(ctx == 0, new)] = 0
    rows = int(pages.sum()) * page
    return dict(case=case, q=_normal(g, (int(new.sum()), qh, hd), TYPES[case["dtype"]]), k_cache=_cache(g, rows, kvh, hd),
                v_cache=_cache(g, rows, kvh, hd), query_seq=_dev(seq), key_len=_dev(key_len), table=_dev(table),
                cu=np.concatenate([[0], np.cumsum(new)]).astype(np.int32), few=int(new.max()) <= 8,
                decode=bool((new == 1).all()))


def _prepare_store(case: dict, g, r) -> dict:
    qh, kvh, hd = HEADS[case["heads"]]
    t, dt = case["tokens"], TYPES[case["dtype"]]
    i = torch.arange(case["rot"] // 2, dtype=torch.float64, device=DEV)
    slots = r.permutation(t + 64)[:t].astype(np.int32)
    slots[3::50] = -1  # tokens that are not stored
    return dict(case=case, qkv=_normal(g, (t, (qh + 2 * kvh) * hd), dt),
                positions=torch.randint(0, case["far"], (t,), generator=g, device=DEV),
                inv_freq=1e6 ** (-2.0 * i / case["rot"]), q_out=torch.empty((t, qh * hd), dtype=dt, device=DEV),
                q_w=_normal(g, (hd,), dt, 1.0, 0.1) if case["norm"] else None,
                k_w=_normal(g, (hd,), dt, 1.0, 0.1) if case["norm"] else None, slots=_dev(slots),
                k_cache=_cache(g, t + 64, kvh, hd), v_cache=_cache(g, t + 64, kvh, hd))


def _prepare_prompt(case: dict, g, r) -> dict:
    qh, kvh, hd = HEADS[case["heads"]]
    cu = np.concatenate([[0], np.cumsum(_ints(case["lens"]))])
    t = int(cu[-1])
    qkv = _normal(g, (t, (qh + 2 * kvh) * hd), TYPES[case["dtype"]]).view(t, qh + 2 * kvh, hd)
    return dict(case=case, q=qkv[:, :qh], k=qkv[:, qh:qh + kvh], v=qkv[:, qh + kvh:], cu=_dev(cu))


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    make = dict(kv4=_prepare_kv4, store=_prepare_store, prompt=_prepare_prompt)
    return make[case["family"]](case, g, np.random.default_rng(seed))


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _pack(x: torch.Tensor) -> torch.Tensor:
    """Values [rows, kvh, hd] (32 or 64 bits) as rows of a 4-bit cache."""
    rows, kvh, hd = x.shape
    x = x.reshape(rows, kvh, hd // GROUP, GROUP)
    low, high = x.amin(-1).clamp_max(0), x.amax(-1).clamp_min(0)
    need = (high - low) / 15
    # the least scale of seven significant bits that is not below
    step = torch.exp2(torch.floor(torch.log2(need.clamp_min(LEAST_NORMAL))) - 6)
    d = (torch.ceil(need / step) * step).clamp_max(MOST_SCALE)
    over = torch.where(d > 0, d, torch.ones_like(d))
    z = torch.round(-low / over).clamp_max(15)
    n = (torch.round(x / over[..., None]) + z[..., None]).clamp(0, 15)
    odd = ~torch.isfinite(x).all(-1)
    n, z = torch.where(odd[..., None], 0.0, n), torch.where(odd, 0.0, z)
    word = d.to(torch.float16).view(torch.int16).int()
    word = torch.where(odd, 0x7E00, word) | z.int()
    n = n.to(torch.uint8).reshape(rows, kvh * hd)
    codes = n[:, 0::2] | (n[:, 1::2] << 4)
    words = torch.stack([word & 255, word >> 8], -1).to(torch.uint8).reshape(rows, -1)
    out = torch.zeros((rows, _row_bytes(kvh, hd)), dtype=torch.uint8, device=x.device)
    out[:, :codes.shape[1]] = codes
    out[:, codes.shape[1]:codes.shape[1] + words.shape[1]] = words
    return out


def _unpack(rows: torch.Tensor, kvh: int, hd: int) -> torch.Tensor:
    """Rows [..., row bytes] of a 4-bit cache as values [..., kvh, hd] in 32 bits."""
    codes = rows[..., :kvh * hd // 2]
    words = rows[..., kvh * hd // 2:kvh * hd // 2 + kvh * (hd // GROUP) * 2].contiguous().view(torch.int16)
    n = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    d = (words & -16).view(torch.float16).float()[..., None]
    z = (words & 15).float()[..., None]
    n = n.view(*rows.shape[:-1], kvh * (hd // GROUP), GROUP)
    return ((n - z) * d).view(*rows.shape[:-1], kvh, hd)


def _softmax_product(scores: torch.Tensor, seen: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
    """softmax over the seen keys (last dim), times v; zeros where none is seen."""
    scores = torch.where(seen, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    return (p @ v) / p.sum(-1, keepdim=True).clamp_min(1e-30)


def _attend_gathered(s: dict) -> torch.Tensor:
    """Each token over the rows of its own sequence."""
    q, page, n = s["q"], s["case"]["page"], s["key_len"].long()[:, None]
    qh, kvh, hd = HEADS[s["case"]["heads"]]
    t = q.shape[0]
    keys = torch.arange(s["table"].shape[1] * page, device=DEV).expand(t, -1)
    seen = keys < n
    entry = s["table"][s["query_seq"].long()[:, None], keys // page]
    rows = torch.where(seen, entry.long() * page + keys % page, torch.zeros_like(keys))
    k = _unpack(s["k_cache"][rows], kvh, hd).permute(0, 2, 3, 1).contiguous()  # [t, kvh, hd, n]
    v = _unpack(s["v_cache"][rows], kvh, hd).permute(0, 2, 1, 3).contiguous()
    scores = (q.float().view(t, kvh, qh // kvh, hd) @ k) * hd ** -0.5
    return _softmax_product(scores, seen[:, None, None, :], v).reshape(t, qh, hd).to(q.dtype)


def _attend_packed(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, seen: torch.Tensor) -> torch.Tensor:
    """q [t, qh, hd] against all keys k, v [n, kvh, hd] (32 bits), of which token t sees seen[t]."""
    t, qh, hd = q.shape
    kvh = k.shape[1]
    g = qh // kvh
    rows = q.float().view(t, kvh, g, hd).permute(1, 2, 0, 3).reshape(kvh, g * t, hd)
    scores = (rows @ k.permute(1, 2, 0).contiguous()) * hd ** -0.5
    out = _softmax_product(scores, seen.repeat(g, 1), v.permute(1, 0, 2).contiguous())
    return out.view(kvh, g, t, hd).permute(2, 0, 1, 3).reshape(t, qh, hd).to(q.dtype)


def _plain_kv4(s: dict) -> torch.Tensor:
    if s["few"]:
        return _attend_gathered(s)
    page = s["case"]["page"]
    _, kvh, hd = HEADS[s["case"]["heads"]]
    entries = s["table"].reshape(-1).long()
    live = (entries >= 0).nonzero().view(-1)
    at = (live[:, None] * page + torch.arange(page, device=DEV)).view(-1)  # (sequence, key) as one number
    width = s["table"].shape[1] * page
    rows = entries[at // page] * page + at % page
    seen = (s["query_seq"].long()[:, None] == at // width) & (at % width < s["key_len"].long()[:, None])
    return _attend_packed(s["q"], _unpack(s["k_cache"][rows], kvh, hd), _unpack(s["v_cache"][rows], kvh, hd), seen)


def _turned(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, w, c: dict) -> torch.Tensor:
    """x [t, heads, hd] with its norm (where there are weights) and rotation, in x's bits."""
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.to(x.dtype)
    r = c["rot"]
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if c["interleaved"] else (x[..., :r // 2], x[..., r // 2:r])
    cos, sin = cos.to(x.dtype)[:, None], sin.to(x.dtype)[:, None]
    y = [a * cos - b * sin, b * cos + a * sin]
    y = torch.stack(y, -1).flatten(-2) if c["interleaved"] else torch.cat(y, -1)
    return torch.cat([y, x[..., r:]], -1)


def _plain_store(s: dict):
    c, qkv = s["case"], s["qkv"]
    qh, kvh, hd = HEADS[c["heads"]]
    t = c["tokens"]
    angle = s["positions"].double()[:, None] * s["inv_freq"]
    cos, sin = torch.cos(angle) * c["scale"], torch.sin(angle) * c["scale"]
    q = _turned(qkv[:, :qh * hd].float().view(t, qh, hd), cos, sin, s["q_w"], c).to(qkv.dtype).view(t, -1)
    # codes change where a value crosses a border between two: 64 bits
    k = _turned(qkv[:, qh * hd:(qh + kvh) * hd].double().view(t, kvh, hd), cos, sin, s["k_w"], c)
    v = qkv[:, (qh + kvh) * hd:].double().view(t, kvh, hd)
    kept = s["slots"] >= 0
    at = s["slots"][kept].long()
    s["k_cache"][at], s["v_cache"][at] = _pack(k)[kept], _pack(v)[kept]
    return q, _unpack(s["k_cache"], kvh, hd).half(), _unpack(s["v_cache"], kvh, hd).half()


def _plain_prompt(s: dict) -> torch.Tensor:
    t = torch.arange(s["q"].shape[0], device=DEV)
    start = s["cu"].long()[torch.searchsorted(s["cu"].long(), t, right=True) - 1]
    seen = (t[None, :] <= t[:, None]) & (t[None, :] >= start[:, None])
    return _attend_packed(s["q"], s["k"].float(), s["v"].float(), seen)


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------
def _run_own(s: dict):
    from nano_vllm_cpp_amd import ops

    c = s["case"]
    qh, kvh, hd = HEADS[c["heads"]]
    if c["family"] == "kv4":
        return ops.paged_attention_kv4(s["q"], s["k_cache"], s["v_cache"], kvh, s["query_seq"], s["key_len"], s["table"],
                                       c["page"], hd ** -0.5, max_query_len=1 if s["decode"] else 0,
                                       cu_seqlens=None if s["decode"] else s["cu"])
    if c["family"] == "prompt":
        return ops.prompt_attention(s["q"], s["k"], s["v"], s["cu"], hd ** -0.5)
    q, k, v = s["qkv"][:, :qh * hd], s["qkv"][:, qh * hd:(qh + kvh) * hd], s["qkv"][:, (qh + kvh) * hd:]
    ops.rotary_store_kv4(q, k, v, s["positions"], s["inv_freq"], qh, kvh, hd, s["k_cache"], s["v_cache"], s["slots"],
                         interleaved=c["interleaved"], attn_scale=c["scale"], q_w=s["q_w"], k_w=s["k_w"], eps=EPS,
                         q_out=s["q_out"])
    return s["q_out"], ops.kv4_unpack(s["k_cache"], kvh, hd), ops.kv4_unpack(s["v_cache"], kvh, hd)


def run(state: dict):
    if own:
        return _run_own(state)
    return dict(kv4=_plain_kv4, store=_plain_store, prompt=_plain_prompt)[state["case"]["family"]](state)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case: dict) -> dict:
    qh, kvh, hd = HEADS[case["heads"]]
    e, row = (4 if case["dtype"] == "f32" else 2), _row_bytes(kvh, hd)
    if case["family"] == "kv4":
        ctx, new = _batch(case)
        pairs = sum(int((np.arange(n - k, n) + 1).sum()) for n, k in zip(ctx, new) if n > 0)
        return dict(bytes=2 * int(ctx.sum()) * row + 2 * int(new.sum()) * qh * hd * e, flops=4.0 * pairs * qh * hd)
    if case["family"] == "store":  # with the caches read back as fp16 values
        t = case["tokens"]
        return dict(bytes=t * ((2 * qh + 2 * kvh) * hd * e + 2 * row) + 2 * (t + 64) * (row + kvh * hd * 2),
                    flops=6.0 * t * (qh + kvh) * hd)
    lens = np.array(_ints(case["lens"]))
    return dict(bytes=int(lens.sum()) * 2 * (qh + kvh) * hd * e, flops=2.0 * int((lens * (lens + 1)).sum()) * qh * hd)


# ---------------------------------------------------------------------------
# the outputs from their definitions, in 64 bits
# ---------------------------------------------------------------------------
def _exact_rows(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, n: torch.Tensor) -> torch.Tensor:
    """q [t, qh, hd] over keys k, v [keys, kvh, hd], of which token t sees the first n[t]."""
    qh, hd = q.shape[1:]
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    later = torch.arange(len(k), device=DEV) >= n[:, None]
    some = n > 0
    for h in range(qh):
        kh = h // (qh // k.shape[1])
        w = q[:, h].double() @ k[:, kh].double().T.contiguous() / math.sqrt(hd)
        w.masked_fill_(later, -math.inf)
        out[some, h] = torch.softmax(w[some], 1) @ v[:, kh].double()
    return out


def _exact_values(rows: torch.Tensor, kvh: int, hd: int) -> torch.Tensor:
    """The values of cache rows, dimension by dimension."""
    out = torch.empty((len(rows), kvh, hd), dtype=torch.float64, device=DEV)
    at = kvh * hd // 2
    for h in range(kvh):
        for i in range(hd):
            byte = rows[:, (h * hd + i) // 2].long()
            n = byte % 16 if i % 2 == 0 else byte // 16
            where = at + 2 * (h * (hd // GROUP) + i // GROUP)
            word = rows[:, where].long() + 256 * rows[:, where + 1].long()
            bits, z = word // 16 * 16, word % 16
            expo, frac = bits // 1024 % 32, bits % 1024
            d = torch.where(expo == 0, frac.double() * 2.0 ** -24, (1024 + frac).double() * 2.0 ** (expo - 25).double())
            out[:, h, i] = (n - z).double() * d
    return out


def _exact_kv4(s: dict) -> torch.Tensor:
    _, kvh, hd = HEADS[s["case"]["heads"]]
    seq, key_len, table = (s[n].cpu().numpy() for n in ("query_seq", "key_len", "table"))
    page = s["case"]["page"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    k_all, v_all = _exact_values(s["k_cache"], kvh, hd), _exact_values(s["v_cache"], kvh, hd)
    for b in np.unique(seq):
        tokens = np.flatnonzero(seq == b)
        j = np.arange(int(key_len[tokens].max()))
        if not len(j):
            continue
        rows = torch.from_numpy(table[b, j // page].astype(np.int64) * page + j % page).to(DEV)
        at = torch.from_numpy(tokens).to(DEV)
        out[at] = _exact_rows(s["q"][at], k_all[rows], v_all[rows], torch.from_numpy(key_len[tokens]).to(DEV))
    return out


def _exact_quantized(x: torch.Tensor) -> torch.Tensor:
    """Each group's values as the cache gives them back."""
    out = torch.empty_like(x)
    powers = torch.tensor([2.0 ** e for e in range(-20, 200)], dtype=torch.float64, device=x.device)
    for i in range(0, x.shape[-1], GROUP):
        part = x[..., i:i + GROUP]
        low, high = torch.minimum(part.min(-1).values, part.new_zeros(())), torch.maximum(part.max(-1).values, part.new_zeros(()))
        frac, expo = torch.frexp((high - low) / 15.0)  # frac in [1/2, 1): seven bits are multiples of 2^-7
        ulp = powers[(expo.long() - 7).clamp_min(-20) + 20]
        d = torch.clamp(torch.ceil((high - low) / 15.0 / ulp) * ulp, max=MOST_SCALE)
        safe = torch.where(d == 0, torch.ones_like(d), d)
        z = torch.clamp(torch.round(low.abs() / safe), max=15.0)
        n = torch.clamp(torch.round(part / safe[..., None]) + z[..., None], 0.0, 15.0)
        out[..., i:i + GROUP] = (n - z[..., None]) * d[..., None]
    return out


def _exact_store(s: dict):
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
    k_cache, v_cache = _exact_values(s["k_cache"], kvh, hd), _exact_values(s["v_cache"], kvh, hd)
    kept = s["slots"] >= 0
    at = s["slots"][kept].long()
    k_cache[at], v_cache[at] = _exact_quantized(y[:, qh:])[kept], _exact_quantized(x[:, qh + kvh:])[kept]
    return y[:, :qh].reshape(t, -1), k_cache, v_cache


def _exact_prompt(s: dict) -> torch.Tensor:
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEV)
    cu = s["cu"].tolist()
    for a, b in zip(cu, cu[1:]):
        out[a:b] = _exact_rows(s["q"][a:b], s["k"][a:b], s["v"][a:b], torch.arange(1, b - a + 1, device=DEV))
    return out


def exact(case: dict, seed: int):
    return dict(kv4=_exact_kv4, store=_exact_store, prompt=_exact_prompt)[case["family"]](prepare(case, seed))
