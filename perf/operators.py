"""The paged-cache attention operators, as cases that can be run and timed.

Three operators of one serving step, over a paged key-value cache
(k_pages, v_pages: [pages][kv_heads][page_size][head_dim]):

  append   q and k normalised per head, rotated by their positions; q returned,
           k and v written to their slots of the cache, in one pass
  decode   attention of each request's newest token(s) over its pages
  prefill  attention of each request's prompt chunk over its pages

`own` False: the operators' plain form, elementary torch operations in 32
bits, rounded once at the end. `own` True: bnn_b200.paged.
"""
import math
import random
import sys
from pathlib import Path

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


# ---- cases

def listed():
    return [
        # One request's next token at the width of the 28-layer benchmark model
        # (16 query heads, 8 KV heads of 128): the smallest call, all latency.
        _append("append_token", tokens=1, src="f32", dtype="bf16"),
        # One step of 61 requests from a 16-bit projection, the rotation on half
        # of each head's dimensions (partial rotary), adjacent pairs.
        _append("append_step_61", tokens=61, src="bf16", dtype="bf16", hq=32, rotary=64, interleaved=True, page=32),
        # A long prompt's chunk straight from the FP32 q|k|v rows of the linears.
        _append("append_prompt_8192", tokens=8192, src="f32", dtype="bf16", page=64),
        # One short conversation: position 160, inside the benchmark's decode range.
        _decode("decode_one_160", batch=1, kv_lo=160, kv_hi=160),
        # Eight contexts at the full 4096-position context.
        _decode("decode_8x4096", batch=8, kv_lo=4096, kv_hi=4096, page=64),
        # Many requests of unlike lengths, from one token to 16 K, 8 query heads per KV head.
        _decode("decode_ragged_61", batch=61, kv_lo=1, kv_hi=16384, key=5, hq=32, hkv=4, dtype="f16"),
        # Two very long documents: few rows, the length has to be split.
        _decode("decode_2x131071", batch=2, kv_lo=131071, kv_hi=131071, page=64, lse=True),
        # Streaming requests: the last 1024 positions and 4 sinks stay visible, older pages were released.
        _decode("decode_window_33", batch=33, kv_lo=700, kv_hi=32768, key=7, hq=16, hkv=2, d=64, window=1024, sinks=4),
        # Eight short prompts entering together (32 to 64 tokens).
        _prefill("prefill_short_8", batch=8, q_lo=32, q_hi=64, ctx_hi=0, key=1),
        # The 512-token prompt of the prefill benchmark.
        _prefill("prefill_512", batch=1, q_lo=512, q_hi=512, ctx_hi=0),
        # A long prompt in one call.
        _prefill("prefill_8192", batch=1, q_lo=8192, q_hi=8192, ctx_hi=0, page=64),
        # Chunks of unlike lengths behind unlike contexts, window and sinks, released pages.
        _prefill("prefill_window_chunks", batch=5, q_lo=300, q_hi=2048, ctx_lo=1000, ctx_hi=12000, key=3, hq=32, hkv=8, d=64,
                 dtype="f16", window=2048, sinks=4, lse=True),
    ]


def _append(name=None, *, tokens, src, dtype, hq=16, hkv=8, d=128, rotary=None, interleaved=False, page=16):
    c = {"op": "append", "tokens": tokens, "src": src, "dtype": dtype, "hq": hq, "hkv": hkv, "d": d,
         "rotary": d if rotary is None else rotary, "interleaved": interleaved, "page": page}
    return dict(c, name=name) if name else c


def _decode(name=None, *, batch, kv_lo, kv_hi, key=0, hq=16, hkv=8, d=128, page=16, dtype="bf16", window=0, sinks=0, new=1,
            lse=False):
    c = {"op": "decode", "batch": batch, "q_lo": new, "q_hi": new, "kv_lo": kv_lo, "kv_hi": kv_hi, "key": key, "hq": hq, "hkv": hkv,
         "d": d, "page": page, "dtype": dtype, "window": window, "sinks": sinks, "lse": lse}
    return dict(c, name=name) if name else c


def _prefill(name=None, *, batch, q_lo, q_hi, ctx_lo=0, ctx_hi, key=0, hq=16, hkv=8, d=128, page=16, dtype="bf16", window=0, sinks=0,
             lse=False):
    c = {"op": "prefill", "batch": batch, "q_lo": q_lo, "q_hi": q_hi, "ctx_lo": ctx_lo, "ctx_hi": ctx_hi, "key": key, "hq": hq,
         "hkv": hkv, "d": d, "page": page, "dtype": dtype, "window": window, "sinks": sinks, "lse": lse}
    return dict(c, name=name) if name else c


def _log_int(rng, lo, hi):
    """An integer of [lo, hi], its logarithm evenly spread."""
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(("append", "decode", "decode", "prefill", "prefill"))
    d = rng.choice((64, 128, 128))
    hkv = rng.choice((1, 2, 4, 8))
    page = rng.choice((16, 32, 64, 128))
    dtype = rng.choice(("bf16", "f16"))
    if op == "append":
        hq = hkv * rng.choice((1, 2, 3, 4, 8))
        return _append(tokens=_log_int(rng, 1, 8192 * 32 * 128 // (d * (hq + 2 * hkv))) if hq + 2 * hkv > 32 else _log_int(rng, 1, 8192),
                       src=rng.choice(("f32", "bf16", "f16")), dtype=dtype, hq=hq, hkv=hkv, d=d, rotary=rng.choice((d, d, d // 2)),
                       interleaved=rng.random() < 0.3, page=page)
    window, sinks = rng.choice(((0, 0), (0, 0), (rng.randrange(64, 4097), rng.randrange(0, 9))))
    if op == "decode":
        group = rng.choice((1, 2, 3, 4, 5, 7, 8))
        hi = _log_int(rng, 16, 131071)
        most = max(1, min(128, 2 * 131071 * 8 * 128 // (hi * hkv * d)))
        new = rng.choice((1, 1, 1, 2))
        return _decode(batch=_log_int(rng, 1, most), kv_lo=_log_int(rng, new, hi), kv_hi=hi, key=rng.randrange(1 << 20), hq=hkv * group,
                       hkv=hkv, d=d, page=page, dtype=dtype, window=window, sinks=sinks, new=new, lse=rng.random() < 0.5)
    hq = hkv * rng.choice([g for g in (1, 2, 3, 4, 8) if g * hkv <= 32])
    hi = _log_int(rng, 24, 4096)
    ctx = rng.choice((0, _log_int(rng, 1, 8192)))
    most = max(1, min(16, 8192 * 8192 * 16 // (2 * hi * (hi + ctx) * hq)))  # padded pairs stay under the largest listed case's
    return _prefill(batch=_log_int(rng, 1, most), q_lo=_log_int(rng, 17, hi), q_hi=hi, ctx_lo=min(ctx, 1), ctx_hi=ctx,
                    key=rng.randrange(1 << 20), hq=hq, hkv=hkv, d=d, page=page, dtype=dtype, window=window, sinks=sinks,
                    lse=rng.random() < 0.5)


def _lengths(case):
    """(new tokens, cache length with them) of each request: they follow from the case alone."""
    r = random.Random(case["key"])
    got = []
    for i in range(case["batch"]):
        n = case["q_hi"] if i == 0 else _log_int(r, case["q_lo"], case["q_hi"])
        if case["op"] == "decode":
            kv = case["kv_hi"] if i == 0 else _log_int(r, case["kv_lo"], case["kv_hi"])
            got.append((n, max(kv, n)))
        else:
            ctx = case["ctx_hi"] if i == 0 or not case["ctx_hi"] else _log_int(r, max(1, case["ctx_lo"]), case["ctx_hi"])
            got.append((n, ctx + n))
    return got


# ---- inputs

def _append_pages(case):
    return -(-case["tokens"] // case["page"]) + 3


def prepare(case, seed):
    return (_prepare_append if case["op"] == "append" else _prepare_attention)(case, seed)


def _prepare_append(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t, hq, hkv, d, page = (case[k] for k in ("tokens", "hq", "hkv", "d", "page"))
    dtype = _DTYPES[case["dtype"]]
    # the linears' rows: each token with a magnitude of its own, a few large channels
    x = torch.randn(t, (hq + 2 * hkv) * d, device="cuda", generator=g)
    x *= 0.5 + 4 * torch.rand(t, 1, device="cuda", generator=g)
    x *= 1 + 8 * (torch.rand(x.shape[1], device="cuda", generator=g) < 0.01)
    most = 16384
    half = case["rotary"] // 2
    angle = torch.arange(most, device="cuda", dtype=torch.float64)[:, None] * \
        1e6 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
    # a prompt's tokens stand one behind another; a step's come from many requests
    first = int(torch.randint(0, most - t + 1, (1,), device="cuda", generator=g))
    positions = first + torch.arange(t, device="cuda") if t > 256 else torch.randint(0, most, (t,), device="cuda", generator=g)
    pages = _append_pages(case)
    slots = torch.randperm(pages, device="cuda", generator=g)[:, None] * page + torch.arange(page, device="cuda")
    slots = slots.reshape(-1)[:t].contiguous()
    if t > 16:
        slots[t // 3] = -1  # a padding token of the batch: not stored
    return {"case": dict(case), "qkv": x.to(_DTYPES[case["src"]]),
            "q_norm": 1 + 0.3 * torch.randn(d, device="cuda", generator=g), "k_norm": 1 + 0.3 * torch.randn(d, device="cuda", generator=g),
            "cos": angle.cos().float(), "sin": angle.sin().float(), "positions": positions.int(), "slots": slots.int(),
            "k_pages": torch.randn(pages, hkv, page, d, device="cuda", generator=g).to(dtype),
            "v_pages": torch.randn(pages, hkv, page, d, device="cuda", generator=g).to(dtype)}


def _used_pages(case, n, kv):
    """The page numbers of one request that a query can still see; the others were released."""
    page, window = case["page"], case["window"]
    last = (kv - 1) // page
    if not window:
        return list(range(last + 1))
    first = max(0, kv - n - window + 1) // page
    sink = [p for p in range(-(-case["sinks"] // page)) if p < first]
    return sink + list(range(first, last + 1))


def _prepare_attention(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    hq, hkv, d, page = (case[k] for k in ("hq", "hkv", "d", "page"))
    dtype = _DTYPES[case["dtype"]]
    lengths = _lengths(case)
    used = [_used_pages(case, n, kv) for n, kv in lengths]
    width = max(-(-kv // page) for _, kv in lengths)
    pages = sum(map(len, used)) + 2
    order = torch.randperm(pages, device="cuda", generator=g)[:pages - 2].int()
    rows = torch.tensor([b * width + p for b, u in enumerate(used) for p in u], device="cuda")
    table = torch.full((len(lengths) * width,), -1, device="cuda", dtype=torch.int32)
    table[rows] = order
    starts = [0]
    for n, _ in lengths:
        starts.append(starts[-1] + n)
    # queries and keys as their norms leave them (unit scale times trained gains)
    q_gain = 1.5 + torch.rand(d, device="cuda", generator=g)
    k_gain = 1 + torch.rand(d, device="cuda", generator=g)
    k = torch.randn(pages, hkv, page, d, device="cuda", generator=g, dtype=torch.float32 if pages * page * hkv * d < 1 << 28 else dtype)
    return {"case": dict(case), "q": (torch.randn(starts[-1], hq, d, device="cuda", generator=g) * q_gain).to(dtype),
            "k_pages": k.mul_(k_gain.to(k.dtype)).to(dtype),
            "v_pages": torch.randn(pages, hkv, page, d, device="cuda", generator=g, dtype=dtype),
            "page_table": table.view(len(lengths), width),
            "kv_lens": torch.tensor([kv for _, kv in lengths], device="cuda", dtype=torch.int32),
            "q_starts": torch.tensor(starts, device="cuda", dtype=torch.int32),
            "max_q": max(n for n, _ in lengths), "max_kv": max(kv for _, kv in lengths)}


# ---- one pass

def run(state):
    if state["case"]["op"] == "append":
        return (_append_own if own else _append_plain)(state)
    return (_attention_own if own else _attention_plain)(state)


_paged = None


def _ops():
    """The operators' handle, made once as a program makes it."""
    global _paged
    if _paged is None:
        at = str(Path(__file__).resolve().parents[1] / "bnn-train-infer_b200")
        if at not in sys.path:
            sys.path.insert(0, at)
        from bnn_b200 import accel, paged
        _paged = paged.Paged(accel.Device(0), max_batch=256)
    return _paged


def _split_heads(state):
    c, x = state["case"], state["qkv"]
    return x.view(x.shape[0], -1, c["d"]).split((c["hq"], c["hkv"], c["hkv"]), dim=1)


def _append_own(state):
    c = state["case"]
    q, k, v = _split_heads(state)
    out = _ops().append(q, k, v, state["cos"], state["sin"], state["positions"], state["slots"], state["k_pages"], state["v_pages"],
                        q_norm=state["q_norm"], k_norm=state["k_norm"], eps=1e-6, interleaved=c["interleaved"])
    return {"q": out, "k_pages": state["k_pages"], "v_pages": state["v_pages"]}


def _attention_own(state):
    c = state["case"]
    got = _ops().attention(state["q"], state["k_pages"], state["v_pages"], state["page_table"], state["kv_lens"], state["q_starts"],
                           max_q=state["max_q"], window=c["window"], sinks=c["sinks"], return_lse=c["lse"])
    return {"out": got[0], "lse": got[1]} if c["lse"] else {"out": got}


def _append_plain(state):
    c = state["case"]
    cos, sin = (state[n][state["positions"].long()][:, None] for n in ("cos", "sin"))

    def turned(x, gain):
        x = x.float()
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * gain
        r = c["rotary"]
        if c["interleaved"]:
            a, b = x[..., 0:r:2], x[..., 1:r:2]
            return torch.cat((torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2), x[..., r:]), -1)
        a, b = x[..., :r // 2], x[..., r // 2:r]
        return torch.cat((a * cos - b * sin, b * cos + a * sin, x[..., r:]), -1)

    q, k, v = _split_heads(state)
    dtype = state["k_pages"].dtype
    kept = torch.nonzero(state["slots"] >= 0)[:, 0]
    slots = state["slots"][kept].long()
    at = (slots // c["page"], slice(None), slots % c["page"])
    state["k_pages"][at] = turned(k, state["k_norm"])[kept].to(dtype)
    state["v_pages"][at] = v[kept].float().to(dtype)
    return {"q": turned(q, state["q_norm"]).to(dtype), "k_pages": state["k_pages"], "v_pages": state["v_pages"]}


def _attention_plain(state):
    c = state["case"]
    hkv, d, page = c["hkv"], c["d"], c["page"]
    q, kv_lens, starts = state["q"], state["kv_lens"].long(), state["q_starts"].long()
    new = starts[1:] - starts[:-1]
    key = torch.arange(state["max_kv"], device=q.device)
    pages = state["page_table"].long()[:, key // page]
    there = (pages >= 0) & (key < kv_lens[:, None])
    at = (pages.clamp(min=0), slice(None), (key % page).expand_as(pages))
    k = state["k_pages"][at].float().transpose(1, 2)  # [request, KV head, key, dim]
    v = torch.where(there[:, :, None, None], state["v_pages"][at].float(), 0).transpose(1, 2)
    i = torch.arange(state["max_q"], device=q.device)
    rows = (starts[:-1, None] + i).clamp(max=q.shape[0] - 1)
    qf = q[rows].float().view(len(new), len(i), hkv, -1, d).permute(0, 2, 3, 1, 4)  # [request, KV head, head of the group, query, dim]
    shape = qf.shape
    s = qf.reshape(shape[0], hkv, -1, d) @ k.transpose(2, 3)
    s = s.view(*shape[:4], -1).mul_(1 / math.sqrt(d))
    del k
    position = (kv_lens - new)[:, None] + i
    seen = there[:, None] & (key <= position[..., None])
    if c["window"]:
        seen &= (key > position[..., None] - c["window"]) | (key < c["sinks"])
    s.masked_fill_(~seen[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    s.sub_(m.clamp(min=torch.finfo(torch.float32).min)).exp_()
    total = s.sum(-1, keepdim=True)
    o = (s.reshape(shape[0], hkv, -1, s.shape[-1]) @ v).view(shape)
    o = torch.where(total > 0, o / total, 0).permute(0, 3, 1, 2, 4).reshape(len(new), len(i), -1, d)
    token = torch.arange(q.shape[0], device=q.device)
    owner = torch.searchsorted(starts, token, right=True) - 1
    got = {"out": o[owner, token - starts[owner]].to(q.dtype)}
    if c["lse"]:
        lse = (m + total.log())[..., 0].permute(0, 3, 1, 2).reshape(len(new), len(i), -1)
        got["lse"] = lse[owner, token - starts[owner]]
    return got


# ---- what a pass cannot do without

def work(case):
    esz = 2
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    if case["op"] == "append":
        values = case["tokens"] * (hq + 2 * hkv) * d
        turned = case["tokens"] * (hq + hkv) * d
        return {"bytes": values * ((4 if case["src"] == "f32" else 2) + esz) + case["tokens"] * (case["rotary"] * 4 + 8) + 8 * d,
                "flops": 6 * turned}
    keys = pairs = tokens = 0
    window, sinks = case["window"], case["sinks"]
    for n, kv in _lengths(case):
        tokens += n
        for p in range(kv - n, kv):
            pairs += p + 1 if not window else min(p + 1, window + max(0, min(sinks, p + 1 - window)))
        low = max(0, kv - n - window + 1) if window else 0
        keys += kv - low + min(sinks, low)
    return {"bytes": 2 * keys * hkv * d * esz + 2 * tokens * hq * d * esz + (4 * tokens * hq if case["lse"] else 0) +
            4 * -(-keys // case["page"]),
            "flops": 4 * pairs * hq * d}


# ---- the definition in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return _append_exact(case, s) if case["op"] == "append" else _attention_exact(case, s)


def _append_exact(case, s):
    d, hq, hkv, half = case["d"], case["hq"], case["hkv"], case["rotary"] // 2
    x = s["qkv"].double().view(-1, hq + 2 * hkv, d)
    gains = torch.cat((s["q_norm"].double().expand(hq, d), s["k_norm"].double().expand(hkv, d)))
    y = x[:, :hq + hkv]
    y = gains * y / torch.sqrt(torch.sum(y ** 2, dim=2, keepdim=True) / d + 1e-6)
    # the rotation as a product of complex numbers
    turn = torch.complex(s["cos"].double(), s["sin"].double())[s["positions"].long()].unsqueeze(1)
    lo = torch.arange(half, device=x.device) * (2 if case["interleaved"] else 1)
    hi = lo + (1 if case["interleaved"] else half)
    z = torch.complex(y[..., lo], y[..., hi]) * turn
    y = y.clone()
    y[..., lo], y[..., hi] = z.real, z.imag
    pools = [s["k_pages"].double(), s["v_pages"].double()]
    for pool, rows in zip(pools, (y[:, hq:], x[:, hq + hkv:])):
        flat = pool.transpose(1, 2).reshape(-1, hkv, d)
        ok = s["slots"] >= 0
        flat[s["slots"][ok].long()] = rows[ok]
        pool.copy_(flat.view(pool.shape[0], case["page"], hkv, d).transpose(1, 2))
    return {"q": y[:, :hq], "k_pages": pools[0], "v_pages": pools[1]}


def _attention_exact(case, s):
    hq, hkv, d, page = (case[k] for k in ("hq", "hkv", "d", "page"))
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device=s["q"].device)
    starts, at = s["q_starts"].tolist(), torch.arange
    for b, kv in enumerate(s["kv_lens"].tolist()):
        n = starts[b + 1] - starts[b]
        j = torch.tensor([p * page + o for p in _used_pages(case, n, kv) for o in range(page) if p * page + o < kv], device=out.device)
        slot = s["page_table"][b].long()[j // page]
        for h in range(hkv):
            k = s["k_pages"][slot, h, j % page].double()
            v = s["v_pages"][slot, h, j % page].double()
            for first in range(0, n, 2048):
                last = min(n, first + 2048)
                pos = kv - n + at(first, last, device=out.device).unsqueeze(1)
                far = (j < case["sinks"]) | (pos - j < case["window"]) if case["window"] else True
                hidden = ~((j <= pos) & far)
                for head in range(h * (hq // hkv), (h + 1) * (hq // hkv)):
                    rows = slice(starts[b] + first, starts[b] + last)
                    score = (s["q"][rows, head].double() @ k.T / math.sqrt(d)).masked_fill(hidden, -math.inf)
                    lse[rows, head] = torch.logsumexp(score, 1)
                    out[rows, head] = torch.exp(score - lse[rows, head].unsqueeze(1)) @ v
    return {"out": out, "lse": lse} if case["lse"] else {"out": out}
