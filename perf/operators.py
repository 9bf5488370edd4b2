"""Measured cases of the quantised key/value cache: writing it (head norms, rotary positions and quantisation in one
pass), reading it back, and attention over it for single tokens, trees of drafted tokens and prompt chunks.

A case is a dict of plain values:
  op      "write" | "read" | "attend"
  fmt     "fp8" (e4m3) | "int8" | "int4": what the cache holds, one scale per token and head (int4: a zero point too)
  B       sequences; T new tokens of each at most (ragged: T * 1/B .. T); ctx_lo .. ctx_hi cached tokens of each
  hq, hkv query / key-value heads; d head size; page tokens per page; half: fp16 instead of bf16
  write:  norm (head norms on / off), rot (rotated channels, 0 = none), inter (interleaved pairs instead of halves)
  attend: tree (a random tree's ancestor mask; else every token sees the new tokens up to itself)
The lengths follow from the case alone, so that `work` can count them; everything else comes from the seed.
"""
import math

import numpy as np
import torch

own = False

EPS = 1e-6
_NO = {"norm": False, "rot": 0, "inter": False, "tree": False, "ragged": False, "half": False}


def _case(name, op, fmt, B, T, ctx_lo, ctx_hi, hq, hkv, d, page, **more):
    return {"name": name, "op": op, "fmt": fmt, "B": B, "T": T, "ctx_lo": ctx_lo, "ctx_hi": ctx_hi, "hq": hq, "hkv": hkv,
            "d": d, "page": page, **_NO, **more}


def listed():
    return [
        # one decode step's new token of one sequence, 64 / 8 heads of 128 (the decoder layer the benchmark runs): latency
        _case("write_one_token", "write", "fp8", 1, 1, 1000, 1000, 64, 8, 128, 64, norm=True, rot=128),
        # a decode batch with short drafts, rotation of half the channels in interleaved pairs, no head norms
        _case("write_drafts_int8", "write", "int8", 61, 5, 100, 3000, 32, 8, 128, 16, rot=64, inter=True, ragged=True),
        # ragged prompts of smaller heads into 4 bits (read back, because packed nibbles are no values)
        _case("write_prompts_int4", "write", "int4", 7, 777, 0, 50, 24, 4, 64, 32, norm=True, rot=64, ragged=True, half=True),
        # a long prompt chunk
        _case("write_prompt_fp8", "write", "fp8", 1, 8192, 0, 0, 64, 8, 128, 64, norm=True, rot=128),
        # a cache read back to 16 bits for code that wants plain tensors
        _case("read_ragged_fp8", "read", "fp8", 5, 0, 33, 2100, 32, 8, 128, 64),
        _case("read_long_int4", "read", "int4", 2, 0, 30001, 65536, 64, 8, 128, 64),
        # decode: one new token of one sequence, short cache: latency
        _case("attend_one_token", "attend", "fp8", 1, 1, 1000, 1000, 64, 8, 128, 64),
        # decode: a batch of different lengths
        _case("attend_batch_fp8", "attend", "fp8", 32, 1, 500, 16000, 64, 8, 128, 64),
        # decode: one long sequence on one of eight GPUs' share of the heads
        _case("attend_long_int8", "attend", "int8", 1, 1, 131000, 131000, 8, 1, 128, 64),
        # verification of small ragged trees, 4-bit cache, small heads and pages
        _case("attend_tree_int4", "attend", "int4", 16, 7, 100, 9000, 32, 8, 64, 16, tree=True, ragged=True, half=True),
        # verification of large trees over long caches
        _case("attend_tree64_fp8", "attend", "fp8", 8, 64, 7000, 16000, 64, 8, 128, 64, tree=True),
        # a chunk of a prompt over what came before it
        _case("attend_chunk_fp8", "attend", "fp8", 1, 1000, 7000, 7000, 64, 8, 128, 64),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        op = rng.choice(["write", "read", "attend", "attend"])
        hkv = rng.choice([1, 2, 4, 8])
        hq = hkv * rng.choice([1, 2, 4, 5, 8])
        d = rng.choice([64, 128, 128])
        page = rng.choice([16, 32, 64, 128, 48])
        fmt = rng.choice(["fp8", "int8", "int4"])
        B = _log(rng, 1, 64)
        more = {"half": rng.random() < 0.3, "ragged": rng.random() < 0.5}
        hi = _log(rng, 1, 100000)
        lo = rng.choice([hi, rng.randint(0, hi)])
        if op == "write":
            T = _log(rng, 1, 8192)
            rot = rng.choice([0, d // 2, d, d])
            more |= {"norm": rng.random() < 0.6, "rot": rot, "inter": rng.random() < 0.3}
            hi = lo = min(hi, 2000)
        elif op == "read":
            T = 0
            more["ragged"] = False
        else:
            tree = rng.random() < 0.5
            T = rng.choice([1, 1, _log(rng, 1, 64), _log(rng, 1, 1000)])
            T = min(T, 100) if tree else T
            more["tree"] = tree and T > 1
        if not more["ragged"]:
            T = max(T, 0)
        c = _case("", op, fmt, B, T, lo, hi, hq, hkv, d, page, **more)
        del c["name"]
        w = work(c)
        if op == "write" and w["bytes"] > 3e8:
            continue
        if op == "read" and w["bytes"] > 2.5e8:
            continue
        if op == "attend" and (w["flops"] > 2.4e11 or w["bytes"] > 6e8 or B * T * hq * (hi + T) > 5e8 or B * (hi + T) * hkv * d > 4e8):
            continue
        return c


def _lens(c):
    """Cached tokens and new tokens of every sequence: spread over their ranges, in a fixed shuffled order."""
    B = c["B"]
    part = (np.arange(B) * 7 + 3) % B if B % 7 else np.arange(B)
    share = np.ones(B) if B == 1 else part / (B - 1)
    ctx = np.round(c["ctx_lo"] + (c["ctx_hi"] - c["ctx_lo"]) * share).astype(np.int64)
    new = np.full(B, c["T"], dtype=np.int64)
    if c["ragged"]:
        new = np.maximum(1, np.ceil(c["T"] * (np.arange(B) * 5 % B + 1) / B)).astype(np.int64)
    return ctx, new


def _row_bytes(c):
    """Bytes of one token and head in the cache: codes, scale and, in 4 bits, the zero point."""
    return c["d"] // 2 + 5 if c["fmt"] == "int4" else c["d"] + 4


def work(case):
    ctx, new = _lens(case)
    d, hq, hkv, n = case["d"], case["hq"], case["hkv"], int(new.sum())
    if case["op"] == "write":
        moved = n * d * 2 * (2 * hq + 2 * hkv) + n * 2 * hkv * _row_bytes(case) + n * case["rot"] * 4
        flops = n * (hq + hkv) * d * ((4 if case["norm"] else 0) + (3 if case["rot"] else 0)) + n * 2 * hkv * d * 3
        if case["fmt"] == "int4":      # read back: the codes once more, and the 16-bit values
            moved += int((ctx + new).sum()) * 2 * hkv * _row_bytes(case) + case["B"] * int((ctx + new).max()) * 2 * hkv * d * 2
        return {"bytes": moved, "flops": flops}
    if case["op"] == "read":
        return {"bytes": int(ctx.sum()) * 2 * hkv * _row_bytes(case) + case["B"] * int(ctx.max()) * 2 * hkv * d * 2,
                "flops": int(ctx.sum()) * 2 * hkv * d}
    seen = (ctx * new).sum() + (new.sum() if case["tree"] else (new * (new + 1) // 2).sum())
    moved = int((ctx + new).sum()) * 2 * hkv * _row_bytes(case) + 2 * n * hq * d * 2
    return {"bytes": moved, "flops": int(4 * seen * hq * d)}


def prepare(case, seed):
    c, dev = case, "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    ctx, new = _lens(c)
    B, d, hq, hkv, ps, n = c["B"], c["d"], c["hq"], c["hkv"], c["page"], int(new.sum())
    dt = torch.float16 if c["half"] else torch.bfloat16
    pages = -(-(ctx + new) // ps)
    width, total = int(pages.max()), int(pages.sum()) + 3

    # every sequence's pages lie scattered over the pool; entries behind its last page point nowhere
    order = torch.randperm(total, generator=g, device=dev).to(torch.int32).cpu().numpy()
    table = np.full((B, width), -1, dtype=np.int32)
    at = 0
    for b in range(B):
        table[b, :pages[b]] = order[at:at + pages[b]]
        at += int(pages[b])
    s = {"case": c, "page_table": torch.from_numpy(table).to(dev), "max_len": int((ctx + new).max()), "max_new": int(new.max()),
         "ctx": torch.from_numpy(ctx.astype(np.int32)).to(dev)}
    s["lens"] = s["ctx"] + torch.from_numpy(new.astype(np.int32)).to(dev)
    offsets = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    s["q_offsets"] = torch.from_numpy(offsets).to(dev)

    # the cache: codes of about normal values; slots that no sequence holds carry NaN, as memory never written may
    wide = d // 2 if c["fmt"] == "int4" else d
    scale = lambda: (torch.rand((total, hkv, ps), generator=g, device=dev) + 0.5) * {"fp8": 3 / 448, "int8": 3 / 127, "int4": 5 / 15}[c["fmt"]]  # noqa: E731
    for w in "kv":
        if c["fmt"] == "fp8":
            codes = (torch.randn((total, hkv, ps, wide), generator=g, device=dev, dtype=torch.bfloat16) * 140).clamp_(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
        elif c["fmt"] == "int8":
            codes = (torch.randn((total, hkv, ps, wide), generator=g, device=dev, dtype=torch.bfloat16) * 40).round_().clamp_(-127, 127).to(torch.int8).view(torch.uint8)
        else:
            codes = torch.randint(0, 256, (total, hkv, ps, wide), generator=g, device=dev, dtype=torch.uint8)
            s[w + "_zeros"] = torch.randint(6, 10, (total, hkv, ps), generator=g, device=dev, dtype=torch.uint8)
        s[w + "_codes"], s[w + "_scales"] = codes, scale()
    used = torch.zeros((total, ps), dtype=torch.bool, device=dev)
    spot = torch.arange(width * ps, device=dev)[None]
    valid = spot < s["lens"][:, None]
    page = s["page_table"].long().gather(1, (spot // ps).expand(B, -1)).clamp(min=0)
    used.view(-1)[(page * ps + spot % ps)[valid]] = True
    for w in "kv":
        s[w + "_scales"].masked_fill_(~used[:, None], math.nan)
        if c["fmt"] == "fp8":
            s[w + "_codes"].masked_fill_(~used[:, None, :, None], 0x7F)

    if c["op"] == "read":
        s["lens"] = s["ctx"]
        return s
    seq = torch.from_numpy(np.repeat(np.arange(B), new)).to(dev)
    step = torch.from_numpy(np.concatenate([np.arange(t) for t in new])).to(dev)
    s["seq"], s["step"] = seq, step
    if c["op"] == "write":
        # what the fused projection of queries, keys and values gives: a few channels are much larger than the others
        qkv = torch.randn((n, (hq + 2 * hkv) * d), generator=g, device=dev, dtype=torch.float32)
        big = 1 + 6 * (torch.rand(qkv.shape[1], generator=g, device=dev) > 0.97)
        qkv = (qkv * big).to(dt)
        s["q"], s["k"], s["v"] = (x.view(n, -1, d) for x in qkv.split([hq * d, hkv * d, hkv * d], 1))
        s["q_norm"] = s["k_norm"] = s["table"] = s["positions"] = None
        if c["norm"]:
            s["q_norm"], s["k_norm"] = ((1 + 0.2 * torch.randn(d, generator=g, device=dev)).to(dt) for _ in "qk")
        s["positions"] = (s["ctx"][seq] + step).to(torch.int32)
        if c["rot"]:
            freq = 500000.0 ** (-torch.arange(0, c["rot"], 2, device=dev, dtype=torch.float64) / c["rot"])
            angle = torch.arange(s["max_len"], device=dev, dtype=torch.float64)[:, None] * freq
            s["table"] = torch.cat([angle.cos(), angle.sin()], 1).float()
        return s
    s["q"] = (torch.randn((n, hq, d), generator=g, device=dev, dtype=torch.float32) * (4.0 / math.sqrt(3.0))).to(dt)
    s["mask"] = None
    if c["tree"]:
        T = int(new.max())
        parent = (torch.rand((B, T), generator=g, device=dev).cpu().numpy() * np.arange(T)).astype(np.int64)
        sees = np.zeros((B, T, T), dtype=bool)
        for i in range(T):                    # a token sees itself and what its parent sees
            if i:
                sees[:, i] = sees[np.arange(B), parent[:, i]]
            sees[:, i, i] = True
        s["mask"] = torch.from_numpy(sees).to(dev)[seq, step].contiguous()
    return s


# ---- the framework's calls ----------------------------------------------------------------------------------------
def _handles(s):
    """The cache and the batch as a serving program keeps them: made once for the buffers."""
    if "handles" not in s:
        from gemlite_b200 import kv_cache
        zeros = {w + "_zeros": s[w + "_zeros"] for w in "kv"} if s["case"]["fmt"] == "int4" else {}
        cache = kv_cache.QuantizedKVCache.from_buffers(s["k_codes"], s["v_codes"], s["k_scales"], s["v_scales"],
                                                       kv_format=s["case"]["fmt"], **zeros)
        batch = kv_cache.KVBatch(s["page_table"], s["ctx"], q_offsets=s["q_offsets"], max_len=s["max_len"], max_new=s["max_new"])
        s["handles"] = cache, batch
    return s["handles"]


def _run_own(s):
    c = s["case"]
    cache, batch = _handles(s)
    dt = torch.float16 if c["half"] else torch.bfloat16
    if c["op"] == "read":
        return list(cache.read(s["page_table"], s["lens"], max_len=s["max_len"], out_dtype=dt))
    if c["op"] == "attend":
        return cache.attend(s["q"], batch, mask=s["mask"])
    q = cache.write(s["q"], s["k"], s["v"], batch, positions=s["positions"], cos_sin=s["table"], q_norm=s["q_norm"],
                    k_norm=s["k_norm"], eps=EPS, interleaved=c["inter"])
    if c["fmt"] == "int4":
        return [q, *cache.read(s["page_table"], s["lens"], max_len=s["max_len"], out_dtype=dt)]
    return [q, *_held(s)]


# ---- the plain forms ----------------------------------------------------------------------------------------------
def _held(s):
    kind = torch.float8_e4m3fn if s["case"]["fmt"] == "fp8" else torch.int8
    return [s["k_codes"].view(kind), s["k_scales"], s["v_codes"].view(kind), s["v_scales"]]


def _normed(x, weight):
    """Root-mean-square norm of every head; the sum of squares in 64 bits, because a code next to a border follows it."""
    if weight is None:
        return x.float()
    mean = (x.double().square().sum(-1, keepdim=True) / x.shape[-1]).float()
    return x.float() * (mean + EPS).sqrt().reciprocal() * weight.float()


def _turned(x, s):
    c = s["case"]
    if not c["rot"]:
        return x
    row = s["table"][s["positions"].long()][:, None]
    half = c["rot"] // 2
    cos, sin = row[..., :half], row[..., half:]
    part, rest = x[..., :c["rot"]], x[..., c["rot"]:]
    if c["inter"]:
        a, b = part[..., 0::2], part[..., 1::2]
        return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), rest], -1)
    a, b = part[..., :half], part[..., half:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)


def _quantised(x, fmt):
    """Codes, scale and zero point of every row (a token's head) of x."""
    if fmt == "int4":
        low, high = x.amin(-1, keepdim=True).clamp(max=0), x.amax(-1, keepdim=True).clamp(min=0)
        scale = ((high - low) / torch.full_like(low, 15)).clamp(min=1e-6)
        zero = (-low / scale).round().clamp(0, 15)
        codes = ((x / scale).round() + zero).clamp(0, 15).to(torch.uint8)
        return codes[..., 0::2] | codes[..., 1::2] << 4, scale[..., 0], zero[..., 0].to(torch.uint8)
    most = x.abs().amax(-1, keepdim=True)
    top = 448.0 if fmt == "fp8" else 127.0
    scale = (most / torch.full_like(most, top)).clamp(min=1e-6)
    codes = (x / scale).clamp(-top, top)
    codes = codes.to(torch.float8_e4m3fn) if fmt == "fp8" else codes.round().to(torch.int8)
    return codes.view(torch.uint8), scale[..., 0], None


def _spots(s, length):
    """Page and place in the page of the first `length` tokens of every sequence, and which of them exist."""
    at = torch.arange(length, device=s["ctx"].device)[None].expand(s["ctx"].shape[0], -1)
    page = s["page_table"].long().gather(1, at // s["case"]["page"])
    return page.clamp(min=0), at % s["case"]["page"], at < s["lens"][:, None]


def _values(s, which, length):
    """What the cache holds of the first `length` tokens: [B, length, heads, d] in 32 bits, zeros behind a sequence's end."""
    page, spot, valid = _spots(s, length)
    codes, scale = s[which + "_codes"][page, :, spot], s[which + "_scales"][page, :, spot][..., None]
    if s["case"]["fmt"] == "fp8":
        x = codes.view(torch.float8_e4m3fn).float()
    elif s["case"]["fmt"] == "int8":
        x = codes.view(torch.int8).float()
    else:
        x = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float() - s[which + "_zeros"][page, :, spot][..., None].float()
    return torch.where(valid[..., None, None], x * scale, torch.zeros((), device=x.device))


def _plain_write(s):
    c = s["case"]
    q = _turned(_normed(s["q"], s["q_norm"]), s).to(s["q"].dtype)
    at = s["ctx"][s["seq"]].long() + s["step"]
    page, spot = s["page_table"][s["seq"], at // c["page"]].long(), at % c["page"]
    for w, x in (("k", _turned(_normed(s["k"], s["k_norm"]), s)), ("v", s["v"].float())):
        codes, scale, zero = _quantised(x, c["fmt"])
        s[w + "_codes"][page, :, spot] = codes
        s[w + "_scales"][page, :, spot] = scale
        if zero is not None:
            s[w + "_zeros"][page, :, spot] = zero
    if c["fmt"] == "int4":
        return [q, _values(s, "k", s["max_len"]).to(q.dtype), _values(s, "v", s["max_len"]).to(q.dtype)]
    return [q, *_held(s)]


def _plain_attend(s):
    c = s["case"]
    B, T, L, G = c["B"], s["max_new"], s["max_len"], c["hq"] // c["hkv"]
    k, v = _values(s, "k", L), _values(s, "v", L)
    q = torch.zeros((B, T, c["hkv"], G, c["d"]), device=k.device)
    q[s["seq"], s["step"]] = s["q"].float().view(-1, c["hkv"], G, c["d"])
    score = torch.einsum("bthgd,blhd->bhgtl", q, k) * (1.0 / math.sqrt(c["d"]))
    at = torch.arange(L, device=k.device)[None] - s["ctx"][:, None]                  # which new token, below 0: cached
    if s["mask"] is None:
        sees = at[:, None] <= torch.arange(T, device=k.device)[None, :, None]
    else:
        mask = torch.zeros((B, T, T), dtype=torch.bool, device=k.device)
        mask[s["seq"], s["step"]] = s["mask"]
        sees = mask.gather(2, at.clamp(0, T - 1)[:, None].expand(B, T, L)) | (at < 0)[:, None]
    sees = sees & (at + s["ctx"][:, None] < s["lens"][:, None])[:, None]
    score = score.masked_fill_(~sees[:, None, None], -math.inf)
    p = (score - score.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)
    out = torch.einsum("bhgtl,blhd->bthgd", p, v)
    return out[s["seq"], s["step"]].reshape(-1, c["hq"], c["d"]).to(s["q"].dtype)


def run(state):
    if own:
        return _run_own(state)
    op = state["case"]["op"]
    if op == "write":
        return _plain_write(state)
    if op == "attend":
        return _plain_attend(state)
    dt = torch.float16 if state["case"]["half"] else torch.bfloat16
    return [_values(state, "k", state["max_len"]).to(dt), _values(state, "v", state["max_len"]).to(dt)]


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------
def _cached64(s, which, b, count):
    """[count, heads, d]: what the cache holds of the first `count` tokens of sequence b, page by page."""
    c, found = s["case"], []
    for i in range(-(-count // c["page"])):
        page = int(s["page_table"][b, i])
        codes, scale = s[which + "_codes"][page], s[which + "_scales"][page].double()
        if c["fmt"] == "int4":
            x = torch.empty((c["hkv"], c["page"], c["d"]), dtype=torch.float64, device=codes.device)
            x[..., 0::2], x[..., 1::2] = codes % 16, codes // 16
            x -= s[which + "_zeros"][page].double()[..., None]
        else:
            x = codes.view(torch.float8_e4m3fn if c["fmt"] == "fp8" else torch.int8).double()
        found.append((x * scale[..., None]).transpose(0, 1))
    return torch.cat(found)[:count] if found else torch.empty((0, c["hkv"], c["d"]), dtype=torch.float64, device="cuda")


def _rotated64(x, weight, s):
    c, x = s["case"], x.double()
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.double()
    if c["rot"]:
        row = s["table"].double()[s["positions"].long()][:, None]
        turn = torch.complex(row[..., :c["rot"] // 2], row[..., c["rot"] // 2:])
        pairs = x[..., :c["rot"]].unflatten(-1, (-1, 2) if c["inter"] else (2, -1))
        pairs = pairs if c["inter"] else pairs.transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        x = torch.cat([(z if c["inter"] else z.transpose(-1, -2)).flatten(-2), x[..., c["rot"]:]], -1)
    return x


def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    lens, ctx = s["lens"].tolist(), s["ctx"].tolist()
    if c["op"] == "read":
        whole = [torch.zeros((c["B"], s["max_len"], c["hkv"], c["d"]), dtype=torch.float64, device="cuda") for _ in "kv"]
        for b in range(c["B"]):
            for x, w in zip(whole, "kv"):
                x[b, :lens[b]] = _cached64(s, w, b, lens[b])
        return whole
    if c["op"] == "write":
        # the rotated queries and the scales; the codes follow 32-bit values next to borders and have no value in 64 bits
        q = _rotated64(s["q"], s["q_norm"], s)
        if c["fmt"] == "int4":
            return [q, None, None]
        at = s["positions"].tolist()
        pt = s["page_table"].tolist()
        rows = torch.tensor([pt[b][p // c["page"]] * c["page"] + p % c["page"] for b, p in zip(s["seq"].tolist(), at)], device="cuda")
        found = [q]
        for w, x in (("k", _rotated64(s["k"], s["k_norm"], s)), ("v", s["v"].double())):
            scale = s[w + "_scales"].double().transpose(1, 2).flatten(0, 1)
            scale[rows] = (x.abs().amax(-1) / (448 if c["fmt"] == "fp8" else 127)).clamp(min=1e-6)
            found += [None, scale.unflatten(0, (-1, c["page"])).transpose(1, 2)]
        return found
    G, first = c["hq"] // c["hkv"], s["q_offsets"].tolist()
    out = torch.empty((first[-1], c["hq"], c["d"]), dtype=torch.float64, device="cuda")
    for b in range(c["B"]):
        k, v = _cached64(s, "k", b, lens[b]), _cached64(s, "v", b, lens[b])
        t = first[b + 1] - first[b]
        sees = torch.ones((t, lens[b]), dtype=torch.bool, device="cuda")
        sees[:, ctx[b]:] = torch.ones((t, t), device="cuda").tril().bool() if s["mask"] is None else s["mask"][first[b]:first[b + 1], :t]
        for h in range(c["hq"]):
            score = s["q"][first[b]:first[b + 1], h].double() @ k[:, h // G].T / math.sqrt(c["d"])
            out[first[b]:first[b + 1], h] = torch.softmax(score.masked_fill(~sees, -math.inf), -1) @ v[:, h // G]
    return out
