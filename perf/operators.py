"""The operators over a paged K/V cache, as cases that can be timed and compared.

A server that keeps its own pages brings each model step's new tokens (one per sequence, or the rows of prompts) through
these calls:

``append``  rotates the new keys (and queries) by their positions and writes keys and values into the pages, in the cache's
            type: fp32, bf16, or 4 bits (e2m1 codes, an e4m3 scale for 16 values, one fp32 scale for the pool). Of a 4-bit
            cache the written rows are read back, as the values that they stand for.
``attend``  attention of the new tokens over the pages: causal, with an optional window of the newest positions and a few
            first positions that stay visible beside it.

Sizes: a head count, K/V head count and head size of the repository's configurations (8 / 8 / 64, 16 / 4 / 128, 4 / 4 / 64) and of
common grouped-query models, one to 256 sequences, one token to some thousands, contexts to 64 K positions.
"""
import math

import numpy as np
import torch

own = False
PAGE = 16


def listed():
    return [
        # ---- append ------------------------------------------------------------------------------------------------
        # one user's next token on the latency configuration: the smallest call, latency is all of it
        _append("append one token", cache="bf16", rows="f32", batch=1, new=1, ctx=301, heads=8, kv_heads=8, hd=64),
        # the next tokens of a full batch of 256 users, bf16 activations into a 4-bit cache
        _append("append batch to 4 bits", cache="fp4", rows="bf16", batch=256, new=1, ctx=1500, ragged=True, heads=16, kv_heads=4, hd=128),
        # prompts of uneven length taken in together by the fp32 configuration
        _append("append prompts fp32", cache="f32", rows="f32", batch=37, new=200, ctx=200, ragged=True, heads=8, kv_heads=8, hd=64),
        # a long document into a 4-bit cache, the second half of its pages already there: the largest append
        _append("append document to 4 bits", cache="fp4", rows="bf16", batch=1, new=16001, ctx=32001, heads=32, kv_heads=8, hd=128),
        # ---- attention with a window and first positions -----------------------------------------------------------
        # one user far into a conversation, fp32 queries as the decode step has them
        _attend("window one user", cache="bf16", rows="f32", batch=1, new=1, ctx=3001, window=1024, sinks=4, heads=16, kv_heads=4, hd=128),
        # a service under load: 64 users at uneven positions of long conversations
        _attend("window batch", cache="bf16", rows="bf16", batch=64, new=1, ctx=12000, ragged=True, window=4096, sinks=4, heads=32, kv_heads=8, hd=128),
        # the fp32 configuration, gated as its model is
        _attend("window batch fp32", cache="f32", rows="f32", batch=24, new=1, ctx=1000, ragged=True, window=333, sinks=1, gate=True, heads=8, kv_heads=8, hd=64),
        # a long prompt: every position attends to the 1024 before it and the first 16
        _attend("window prompt", cache="bf16", rows="bf16", batch=1, new=8001, ctx=8001, window=1024, sinks=16, heads=16, kv_heads=4, hd=128),
        # a mixed batch: prompts of 1 to 700 tokens on contexts of uneven length, no window
        _attend("mixed prompts", cache="bf16", rows="bf16", batch=13, new=700, ctx=1500, ragged=True, heads=8, kv_heads=8, hd=64),
        # ---- attention over a cache of 4 bits ------------------------------------------------------------------------
        # one user with a very long context
        _attend("4 bits one user", cache="fp4", rows="f32", batch=1, new=1, ctx=65000, heads=16, kv_heads=4, hd=128),
        # 128 users at uneven positions
        _attend("4 bits batch", cache="fp4", rows="bf16", batch=128, new=1, ctx=8000, ragged=True, heads=32, kv_heads=8, hd=128),
        # a chunk of a long prompt over the context so far
        _attend("4 bits prompt chunk", cache="fp4", rows="bf16", batch=1, new=2048, ctx=10001, heads=16, kv_heads=4, hd=128),
    ]


def _append(name, **c):
    return {"name": name, "op": "append", "ragged": False, "window": 0, "sinks": 0, "gate": False, **c}


def _attend(name, **c):
    return {"name": name, "op": "attend", "ragged": False, "window": 0, "sinks": 0, "gate": False, **c}


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """Another call of the same ranges: steps of 1 to 256 sequences, or prompts of up to some thousand tokens, on contexts
    of one position to 64 K, with or without a window, in each pair of types."""
    heads, kv_heads, hd = rng.choice([(8, 8, 64), (16, 4, 128), (4, 4, 64), (32, 8, 128), (14, 2, 64), (12, 2, 128), (8, 1, 128), (16, 2, 64)])
    cache, rows = rng.choice([("bf16", "f32"), ("bf16", "bf16"), ("f32", "f32"), ("fp4", "f32"), ("fp4", "bf16")])
    c = {"op": rng.choice(["append", "attend", "attend"]), "cache": cache, "rows": rows, "heads": heads, "kv_heads": kv_heads, "hd": hd,
         "ragged": rng.random() < 0.6, "gate": False, "window": 0, "sinks": 0}
    if rng.random() < 0.6 or c["op"] == "append" and rng.random() < 0.4:                      # a step
        c["batch"] = _log_int(rng, 1, 256)
        c["new"] = 1
        c["ctx"] = _log_int(rng, 1, min(65000, 2 * 10 ** 8 // (c["batch"] * kv_heads * hd)))
    else:                                                                                     # prompts
        c["batch"] = _log_int(rng, 1, 16)
        most = min(8000, 16000 // c["batch"]) if c["op"] == "append" or rows == "bf16" else 1000 // c["batch"] + 16
        c["new"] = _log_int(rng, 2, most)
        c["ctx"] = c["new"] if rng.random() < 0.5 else c["new"] + _log_int(rng, 1, 2000)
        while c["op"] == "attend" and c["batch"] * c["new"] * c["ctx"] * heads > 1.0e9:      # not over the largest listed call
            c["new"], c["ctx"] = max(1, c["new"] // 2), max(1, c["ctx"] // 2)
    if c["op"] == "attend":
        if rng.random() < 0.6:
            c["window"] = _log_int(rng, 1, 5000)
            c["sinks"] = rng.choice([0, 1, 4, 5, 16, 33])
        c["gate"] = rng.random() < 0.2
    return c


# ---- a call's inputs ------------------------------------------------------------------------------------------------
def _lengths(case):
    """(new tokens, cached positions with them) of each sequence, a matter of the case and not of the seed."""
    B, n, ctx = case["batch"], case["new"], case["ctx"]
    if not case["ragged"]:
        return np.full(B, n), np.full(B, ctx)
    rng = np.random.default_rng(B * 1000003 + n * 1009 + ctx)
    new = rng.integers(1, n + 1, size=B)
    lens = np.maximum(new, rng.integers(1, ctx + 1, size=B))
    new[B // 2], lens[B // 2] = n, ctx                                # one of the longest
    return new, lens


_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def _rope_table(length, hd, base=10000.0):
    """[length][hd] fp32, (cos, sin) of each pair of dims side by side; the angles in 64 bits."""
    inv = base ** (-torch.arange(0, hd, 2, device="cuda", dtype=torch.float64) / hd)
    ang = torch.arange(length, device="cuda", dtype=torch.float64)[:, None] * inv
    return torch.stack([ang.cos(), ang.sin()], dim=-1).reshape(length, hd).float()


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    B, H, KH, D, cache, dt = case["batch"], case["heads"], case["kv_heads"], case["hd"], case["cache"], _TYPES[case["rows"]]
    new, lens = _lengths(case)
    T = int(new.sum())
    need = (lens + PAGE - 1) // PAGE
    pages, most = int(need.sum()) + 3, int(need.max())
    randn = lambda *shape: torch.randn(shape, device="cuda", generator=g)  # noqa: E731
    # pages of the sequences lie anywhere in the pool
    ids = torch.randperm(pages, device="cuda", generator=g).int()
    table = torch.zeros(B, most, dtype=torch.int32, device="cuda")
    at = torch.arange(most, device="cuda")[None] + torch.tensor(np.concatenate([[0], need.cumsum()[:-1]]), device="cuda")[:, None]
    held = torch.arange(most, device="cuda")[None] < torch.tensor(need, device="cuda")[:, None]
    table[held] = ids[at[held]]
    s = {"case": case, "rows": T, "most_new": int(new.max()), "most_len": int(lens.max()), "page_table": table,
         "row_start": torch.tensor(np.concatenate([[0], new.cumsum()]), dtype=torch.int32, device="cuda"),
         "kv_lens": torch.tensor(lens, dtype=torch.int32, device="cuda"), "k_scale": 1.0, "v_scale": 1.0, "kscale": None, "vscale": None}
    # some dims of keys are larger than the rest by a factor, as they are in trained models
    loud = 1.0 + 4.0 * (torch.rand(KH, D, device="cuda", generator=g) < 0.05)
    if cache == "fp4":
        s["k_scale"], s["v_scale"] = 0.021, 0.0083
        for one, scale, by in (("k", s["k_scale"], loud), ("v", s["v_scale"], torch.ones_like(loud))):
            codes = torch.empty(pages, KH, PAGE, D // 2, dtype=torch.uint8, device="cuda")
            scales = torch.empty(pages, KH, PAGE, D // 16, dtype=torch.float8_e4m3fn, device="cuda")
            step = max(1, (1 << 26) // (KH * PAGE * D))
            for p in range(0, pages, step):
                x = randn(min(step, pages - p), KH, PAGE, D) * by[:, None]
                codes[p:p + step], scales[p:p + step] = _to_fp4(x, scale)
            s[one + "pool"], s[one + "scale"] = codes, scales
            s[one + "_scale"] = scale
    else:
        s["kpool"] = (randn(pages, KH, PAGE, D) * loud[:, None]).to(_TYPES[cache])
        s["vpool"] = randn(pages, KH, PAGE, D).to(_TYPES[cache])
    s["q"] = randn(T, H * D).to(dt)
    s["gate"] = torch.rand(T, H * D, device="cuda", generator=g) if case["gate"] else None
    if case["op"] == "append":
        s["k"] = (randn(T, KH, D) * loud).to(dt).reshape(T, KH * D)
        s["v"] = randn(T, KH * D).to(dt)
        s["rope"] = _rope_table(s["most_len"], D)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        from mini_llm_cuda_b200 import api
        s["ops"] = api.Ops(device=0)
        s["cache"] = api.PagedKV(s["kpool"], s["vpool"], s["page_table"], kscale=s["kscale"], vscale=s["vscale"], k_scale=s["k_scale"], v_scale=s["v_scale"])
        s["batch"] = api.NewRows(s["kv_lens"], s["rows"], row_start=s["row_start"] if case["new"] > 1 else None, max_rows=s["most_new"])
        s["out"] = torch.empty_like(s["q"])
        if case["cache"] == "fp4" and case["op"] == "append":
            s["k_out"], s["v_out"] = torch.empty_like(s["k"]), torch.empty_like(s["v"])
    return s


def run(s):
    case = s["case"]
    if own:
        stream = torch.cuda.current_stream().cuda_stream
        if case["op"] == "attend":
            s["ops"].attn_paged(s["cache"], s["batch"], s["q"], s["out"], heads=case["heads"], gate=s["gate"], window=case["window"], sinks=case["sinks"], stream=stream)
            return s["out"]
        s["ops"].kv_append(s["cache"], s["batch"], s["k"], s["v"], rope=s["rope"], q=s["q"], q_out=s["out"], heads=case["heads"], stream=stream)
        if case["cache"] != "fp4":
            return {"q": s["out"], "k": s["kpool"], "v": s["vpool"]}
        s["ops"].kv_read(s["cache"], s["batch"], s["k_out"], s["v_out"], stream=stream)
        return {"q": s["out"], "k": s["k_out"], "v": s["v_out"]}
    return _attend_plain(s) if case["op"] == "attend" else _append_plain(s)


# ---- plain forms ------------------------------------------------------------------------------------------------------
# e2m1: a sign, two bits of exponent, one of mantissa
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _to_fp4(x, pool_scale):
    """Codes (low half of a byte: the even dim) and e4m3 scales of x [..., D] in fp32: for 16 values a scale of
    max|x| / (6 pool_scale), rounded to e4m3 (at most 448), then x / (scale pool_scale) to the nearest code, ties to the even one."""
    x = x.float()
    b = x.reshape(*x.shape[:-1], x.shape[-1] // 16, 16)
    # the host's two scale factors are rounded to fp32 before the tensors see them, every operation below rounds once
    six = float(np.float32(6.0) * np.float32(pool_scale))
    ratio = b.abs().amax(-1) / torch.full((), six, device=x.device)
    scale = ratio.clamp(max=448.0).to(torch.float8_e4m3fn)
    unit = scale.float() * torch.full((), float(np.float32(pool_scale)), device=x.device)
    inv = torch.where(unit > 0, 1.0 / unit, torch.zeros_like(unit))
    y = b * inv[..., None]
    a = y.abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)) | (torch.signbit(y).to(torch.uint8) << 3)
    code = code.reshape(x.shape)
    return code[..., 0::2] | (code[..., 1::2] << 4), scale.reshape(*x.shape[:-1], -1)


def _from_fp4(codes, scales, pool_scale):
    """The values of codes [..., D / 2] and scales [..., D / 16], in fp32."""
    values = torch.tensor(_E2M1 + tuple(-v for v in _E2M1), device=codes.device)
    pairs = torch.stack([values.repeat(16), values.repeat_interleave(16)], dim=1)          # [byte][low, high]
    x = pairs[codes.int()].reshape(*scales.shape, 16)
    return (x * scales.float()[..., None] * torch.full((), float(np.float32(pool_scale)), device=codes.device)).reshape(*codes.shape[:-1], -1)


def _rotate(x, cs):
    """x [T][heads][D], cs [T][D] (cos, sin): dims 2i and 2i + 1 turned by the angle of pair i."""
    c, s = cs[:, None, 0::2], cs[:, None, 1::2]
    a, b = x[..., 0::2].float(), x[..., 1::2].float()
    return torch.stack([c * a - s * b, s * a + c * b], dim=-1).flatten(-2)


def _places(s):
    """Sequence and position of every row, and each row's number in its sequence."""
    start, lens = s["row_start"].long(), s["kv_lens"].long()
    t = torch.arange(s["rows"], device="cuda")
    seq = torch.searchsorted(start, t, right=True) - 1
    i = t - start[seq]
    return seq, i, lens[seq] - (start[seq + 1] - start[seq]) + i


def _append_plain(s):
    case = s["case"]
    KH, H, D, dt = case["kv_heads"], case["heads"], case["hd"], _TYPES[case["rows"]]
    seq, _, pos = _places(s)
    page, slot = s["page_table"].long()[seq, pos // PAGE], pos % PAGE
    cs = s["rope"][pos]
    q = _rotate(s["q"].reshape(-1, H, D), cs).to(dt).flatten(1)
    k, v = _rotate(s["k"].reshape(-1, KH, D), cs), s["v"].reshape(-1, KH, D).float()
    if case["cache"] != "fp4":
        s["kpool"][page, :, slot] = k.to(s["kpool"].dtype)
        s["vpool"][page, :, slot] = v.to(s["vpool"].dtype)
        return {"q": q, "k": s["kpool"], "v": s["vpool"]}
    for x, one in ((k, "k"), (v, "v")):
        codes, scales = _to_fp4(x, s[one + "_scale"])
        s[one + "pool"][page, :, slot] = codes
        s[one + "scale"].view(torch.uint8)[page, :, slot] = scales.view(torch.uint8)
    read = lambda one: _from_fp4(s[one + "pool"][page, :, slot], s[one + "scale"].view(torch.uint8)[page, :, slot].view(torch.float8_e4m3fn), s[one + "_scale"])  # noqa: E731
    return {"q": q, "k": read("k").to(dt).flatten(1), "v": read("v").to(dt).flatten(1)}


def _cached(s, one, pages):
    """Rows of the cache of every sequence, [batch][kv_heads][positions][D] in fp32."""
    table = s["page_table"][:, :pages].long()
    if s["case"]["cache"] == "fp4":
        scales = s[one + "scale"].view(torch.uint8)[table].view(torch.float8_e4m3fn)
        x = _from_fp4(s[one + "pool"][table], scales, s[one + "_scale"])
    else:
        x = s[one + "pool"][table].float()
    return x.permute(0, 2, 1, 3, 4).flatten(2, 3)


def _attend_plain(s):
    case = s["case"]
    B, KH, H, D, n, L = case["batch"], case["kv_heads"], case["heads"], case["hd"], s["most_new"], s["most_len"]
    G = H // KH
    seq, i, _ = _places(s)
    start, lens = s["row_start"].long(), s["kv_lens"].long()
    pages = (L + PAGE - 1) // PAGE
    q = torch.zeros(B, n, KH, G, D, device="cuda")
    q[seq, i] = s["q"].reshape(-1, KH, G, D).float()
    k = _cached(s, "k", pages)
    x = torch.matmul(q.permute(0, 2, 1, 3, 4).reshape(B, KH, n * G, D), k.transpose(-1, -2))
    del k
    x = x.reshape(B, KH, n, G, -1).mul_(1.0 / math.sqrt(D))
    # row i of a sequence stands at position p and sees key j
    p = (lens - (start[1:] - start[:-1]))[:, None] + torch.arange(n, device="cuda")
    j = torch.arange(pages * PAGE, device="cuda")
    sees = j <= p[..., None]
    if case["window"]:
        sees &= (j > p[..., None] - case["window"]) | (j < case["sinks"])
    x.masked_fill_(~sees[:, None, :, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    x = x.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x.reshape(B, KH, n * G, -1), _cached(s, "v", pages)).reshape(B, KH, n, G, D) / torch.where(total == 0, torch.ones_like(total), total)
    o = o.permute(0, 2, 1, 3, 4)[seq, i].flatten(1)
    if s["gate"] is not None:
        o = o * s["gate"]
    return o.to(_TYPES[case["rows"]])


# ---- the same in 64 bits ----------------------------------------------------------------------------------------------
def exact(case, seed):
    """From the definitions, one sequence and K/V head after another. What a 4-bit append stores has no 64-bit value: its codes
    are those of the fp32 arithmetic."""
    s = _inputs(case, seed)
    new, lens = _lengths(case)
    H, KH, D = case["heads"], case["kv_heads"], case["hd"]
    G, first = H // KH, np.concatenate([[0], new.cumsum()])
    if case["op"] == "append":
        pos = torch.cat([torch.arange(L - n, L, device="cuda") for n, L in zip(new.tolist(), lens.tolist())])
        ang = torch.complex(s["rope"].double()[:, 0::2], s["rope"].double()[:, 1::2])[pos][:, None]
        turn = lambda x, h: torch.view_as_real(torch.view_as_complex(x.double().reshape(-1, h, D // 2, 2)) * ang).flatten(1)  # noqa: E731
        q = turn(s["q"], H)
        if case["cache"] == "fp4":
            return {"q": q, "k": None, "v": None}
        pools = {"q": q, "k": s["kpool"].double(), "v": s["vpool"].double()}
        k, v = turn(s["k"], KH).reshape(-1, KH, D), s["v"].double().reshape(-1, KH, D)
        at = 0
        table = s["page_table"].cpu().numpy()
        flat_k, flat_v = pools["k"].permute(0, 2, 1, 3).reshape(-1, KH, D).clone(), pools["v"].permute(0, 2, 1, 3).reshape(-1, KH, D).clone()
        where = np.concatenate([table[b][np.arange(L - n, L) // PAGE].astype(np.int64) * PAGE + np.arange(L - n, L) % PAGE for b, (n, L) in enumerate(zip(new, lens))])
        where = torch.from_numpy(where).cuda()
        flat_k[where], flat_v[where] = k, v
        back = lambda f: f.reshape(-1, PAGE, KH, D).permute(0, 2, 1, 3).contiguous()  # noqa: E731
        return {"q": q, "k": back(flat_k), "v": back(flat_v)}
    if float(sum(n * L for n, L in zip(new.tolist(), lens.tolist()))) * H * D > 4e12:
        return None
    values = torch.tensor([m * sign for sign in (1.0, -1.0) for m in _E2M1], dtype=torch.float64, device="cuda")
    out = torch.zeros(s["rows"], H, D, dtype=torch.float64, device="cuda")

    def rows_of(one, ids, h, L):
        if case["cache"] != "fp4":
            return s[one + "pool"][ids, h].double().reshape(-1, D)[:L]
        c = s[one + "pool"][ids, h].reshape(-1, D // 2)[:L].long()
        v = torch.stack([values[c & 15], values[c >> 4]], dim=-1).reshape(-1, D // 16, 16)
        sc = s[one + "scale"].view(torch.uint8)[ids, h].view(torch.float8_e4m3fn).double().reshape(-1, D // 16, 1)[:L]
        return (v * sc * float(np.float32(s[one + "_scale"]))).reshape(-1, D)

    for b, (n, L) in enumerate(zip(new.tolist(), lens.tolist())):
        ids = s["page_table"][b, :(L + PAGE - 1) // PAGE].long()
        t0 = int(first[b])
        for h in range(KH):
            k, v = rows_of("k", ids, h, L), rows_of("v", ids, h, L)
            for r in range(0, n, 1024):
                m = min(1024, n - r)
                p = torch.arange(L - n + r, L - n + r + m, device="cuda")[:, None, None]
                j = torch.arange(L, device="cuda")
                hidden = j > p
                if case["window"]:
                    hidden = hidden | ((p - j >= case["window"]) & (j >= case["sinks"]))
                q = s["q"][t0 + r:t0 + r + m].double().reshape(m, H, D)[:, h * G:(h + 1) * G]
                w = torch.softmax((q @ k.T / math.sqrt(D)).masked_fill(hidden, -math.inf), dim=-1)
                out[t0 + r:t0 + r + m, h * G:(h + 1) * G] = w @ v
    out = out.flatten(1)
    return out if s["gate"] is None else out * s["gate"].double()


# ---- what a call cannot do without ------------------------------------------------------------------------------------
def work(case):
    """Every new row read and written once, every position of the cache that some row sees read once (its page id with it), the (cos, sin) row
    of every new position; four flops per attended position, query head and dim, three per rotated value."""
    new, lens = _lengths(case)
    H, KH, D = case["heads"], case["kv_heads"], case["hd"]
    e = 4 if case["rows"] == "f32" else 2
    row = KH * D * {"f32": 4, "bf16": 2, "fp4": 0.5625}[case["cache"]]                        # a position's K, or V
    T = int(new.sum())
    if case["op"] == "append":
        n_bytes = T * (2 * H * D * e + 2 * KH * D * e + 2 * row + 4 * D)
        if case["cache"] == "fp4":
            n_bytes += T * 2 * (row + KH * D * e)                                             # read back
        return {"bytes": n_bytes, "flops": 3.0 * T * (H + KH) * D}
    held = attended = 0.0
    for n, L in zip(new.tolist(), lens.tolist()):
        p = np.arange(L - n, L)
        w, k = case["window"], case["sinks"]
        seen = p + 1 if not w else np.minimum(p + 1, np.minimum(w, p + 1) + np.minimum(k, np.maximum(0, p + 1 - w)))
        attended += float(seen.sum())
        low = 0 if not w else max(0, L - n - w + 1)                                           # the first row's window
        held += L - low + min(k, low)
    n_bytes = 2 * T * H * D * e + (4 * T * H * D if case["gate"] else 0) + 2 * held * row + 4 * held / PAGE
    return {"bytes": n_bytes, "flops": 4.0 * attended * H * D}
