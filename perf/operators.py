"""The token-decoding operators as a measurement sees them: their cases, inputs, plain forms and
exact values.

Four operators of one decoder layer that generates a token at a time over a batch:

  norm    root-mean-square norm of x + residual, the sum kept, the output in e4m3 with one scale
          per row (or in the input's type);
  linear  y = x . W^T for few rows of x, W in 4 bits with a scale (and a zero point) per group of
          inputs, x in 16 bits or in e4m3 with a scale per row;
  append  rotary embedding of the new queries and keys, and the new keys and values written to
          their slots of a paged cache (16 bits, or e4m3 with a scale per head);
  attend  attention of one new token per sequence over that cache, heads of the cache shared by
          groups of query heads, all tokens or a sliding window and the first few (sinks).
"""
import math

import torch

own = False

_T = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32,
      "e4m3": torch.float8_e4m3fn}
_SIZE = {"bf16": 2, "f16": 2, "f32": 4, "e4m3": 1}
E4M3_MAX = 448.0
EPS = 1e-6


# ------------------------------------------------------------------------------- the cases
def listed():
    return [
        # one token of one sequence between two linears of a layer: latency
        dict(name="norm_token", op="norm", rows=1, n=4096, dtype="bf16", fp8=True, residual=True),
        # a prompt's rows through the same norm: memory bandwidth
        dict(name="norm_prompt", op="norm", rows=8192, n=5120, dtype="bf16", fp8=True,
             residual=True),
        # rows of an odd width in 32 bits, as a small unaligned head has them
        dict(name="norm_odd", op="norm", rows=771, n=2051, dtype="f32", fp8=False, residual=True),
        # a square projection for one token: the smallest weight read
        dict(name="linear_token", op="linear", m=1, n=4096, k=4096, group=128, zeros=False,
             dtype="bf16", out="bf16"),
        # gate and up of a feed-forward, stacked, for four tokens that the norm left in e4m3
        dict(name="linear_ffn_e4m3", op="linear", m=4, n=27648, k=5120, group=64, zeros=True,
             dtype="e4m3", out="bf16"),
        # the feed-forward's way back for a ragged batch, the finest groups
        dict(name="linear_batch", op="linear", m=13, n=5120, k=13824, group=32, zeros=False,
             dtype="f16", out="f16"),
        # one new token for each of 32 sequences
        dict(name="append_tokens", op="append", seqs=32, chunk=1, start=4095, hq=32, hkv=8, d=128,
             page=64, dtype="bf16", cache="bf16"),
        # prompts of odd length written into an e4m3 cache, from the middle of a page on
        dict(name="append_prompt", op="append", seqs=3, chunk=2731, start=37, hq=40, hkv=8, d=128,
             page=16, dtype="bf16", cache="e4m3"),
        # a single sequence whose length ends one past a page: latency, split over the length
        dict(name="attend_single", op="attend", seqs=1, len_lo=4097, len_hi=4097, hq=40, hkv=8,
             d=128, page=16, dtype="bf16", cache="bf16", window=0, sinks=0),
        # a serving batch of ragged lengths
        dict(name="attend_batch", op="attend", seqs=32, len_lo=1, len_hi=8192, hq=32, hkv=8, d=128,
             page=64, dtype="bf16", cache="bf16", window=0, sinks=0),
        # few long sequences over an e4m3 cache
        dict(name="attend_long_e4m3", op="attend", seqs=4, len_lo=50001, len_hi=65536, hq=64,
             hkv=8, d=128, page=32, dtype="bf16", cache="e4m3", window=0, sinks=0),
        # a sliding window with four sinks, a cache head for every query head
        dict(name="attend_window", op="attend", seqs=64, len_lo=900, len_hi=6000, hq=12, hkv=12,
             d=64, page=16, dtype="f16", cache="f16", window=1024, sinks=4),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "linear", "append", "attend"])
    if op == "norm":
        n = _log(rng, 64, 16384)
        n = n if rng.random() < 0.4 else max(8, n // 8 * 8)
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        most = 8192 * 5120 * 7 // (n * (3 * _SIZE[dtype] + 1))
        return dict(op=op, rows=_log(rng, 1, min(8192, most)), n=n, dtype=dtype,
                    fp8=rng.random() < 0.6, residual=rng.random() < 0.7)
    if op == "linear":
        group = rng.choice([32, 64, 128])
        k = max(group, _log(rng, 256, 28672) // group * group)
        n = _log(rng, 64, min(28672, 27648 * 5120 // k))
        n = n if rng.random() < 0.4 else max(16, n // 16 * 16)
        dtype = rng.choice(["bf16", "f16", "e4m3"])
        out = rng.choice(["bf16", "f16"]) if dtype == "e4m3" else dtype
        return dict(op=op, m=_log(rng, 1, 32), n=n, k=k, group=group, zeros=rng.random() < 0.5,
                    dtype=dtype, out=out)
    hkv = rng.choice([1, 2, 4, 8, 12])
    hq = hkv * rng.choice([1, 2, 4, 5, 7, 8, 16])
    d = rng.choice([64, 128, 128, 96, 256])
    page = rng.choice([16, 32, 64, 128, 24])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    cache = dtype if rng.random() < 0.65 else "e4m3"
    if op == "append":
        most = max(1, 8192 * 56 * 128 // ((hq + 2 * hkv) * d))
        tokens = _log(rng, 1, min(8192, most))
        seqs = _log(rng, 1, min(64, tokens))
        return dict(op=op, seqs=seqs, chunk=tokens // seqs, start=_log(rng, 1, 4096), hq=hq,
                    hkv=hkv, d=d, page=page, dtype=dtype, cache=cache)
    window = _log(rng, 16, 4096) if rng.random() < 0.4 else 0
    seqs = _log(rng, 1, 64)
    most = 32 * 4096 * 8 * 128 // (seqs * hkv * d)
    hi = _log(rng, 16, max(16, min(65536, most)))
    return dict(op=op, seqs=seqs, len_lo=_log(rng, 1, hi), len_hi=hi, hq=hq, hkv=hkv, d=d,
                page=page, dtype=dtype, cache=cache, window=window,
                sinks=rng.choice([0, 1, 4, 16]) if window else 0)


def _lengths(case):
    b = case["seqs"]
    lo, hi = case["len_lo"], case["len_hi"]
    return [hi if b == 1 else lo + (hi - lo) * i // (b - 1) for i in range(b)]


def _visible(case):
    w, s = case["window"], case["sinks"]
    return [n if not w or n <= w else w + min(s, n - w) for n in _lengths(case)]


def work(case):
    op = case["op"]
    if op == "norm":
        rows, n, e = case["rows"], case["n"], _SIZE[case["dtype"]]
        per = e + (2 * e if case["residual"] else 0) + (1 if case["fp8"] else e)
        return {"bytes": rows * n * per + n * e + (4 * rows if case["fp8"] else 0),
                "flops": rows * n * (5 if case["fp8"] else 4)}
    if op == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        per_group = 2 + (1 if case["zeros"] else 0)
        xb = m * k * _SIZE[case["dtype"]] + (4 * m if case["dtype"] == "e4m3" else 0)
        return {"bytes": n * k // 2 + n * (k // case["group"]) * per_group + xb
                + m * n * _SIZE[case["out"]], "flops": 2 * m * n * k}
    e, c = _SIZE[case["dtype"]], _SIZE[case["cache"]]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    if op == "append":
        t = case["seqs"] * case["chunk"]
        return {"bytes": t * d * (2 * hq * e + 2 * hkv * (e + c)) + 8 * t
                + min(t, case["start"] + 2 * case["chunk"]) * d * 4,
                "flops": t * d * (hq + hkv) * 3}
    vis = sum(_visible(case))
    return {"bytes": 2 * vis * hkv * d * c + 2 * case["seqs"] * hq * d * e
            + 4 * sum(-(-v // case["page"]) for v in _visible(case)),
            "flops": 4 * vis * hq * d}


# ------------------------------------------------------------------------------- the inputs
def _pages(lens, page, g):
    """A block table [len(lens), widest] over shuffled pages, -1 past each sequence's last one."""
    need = [-(-n // page) for n in lens]
    total = sum(need) + 3
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    col = torch.arange(max(need), device="cuda")[None, :]
    cnt = torch.tensor(need, device="cuda")
    at = (torch.cumsum(cnt, 0) - cnt)[:, None] + col
    table = torch.where(col < cnt[:, None], order[at.clamp(max=total - 1)], -1).to(torch.int32)
    return table.contiguous(), total


def _cache_fill(shape, kind, scale, g):
    v = torch.randn(shape, generator=g, device="cuda", dtype=torch.float16)
    if kind != "e4m3":
        return v.to(_T[kind])
    return v.div_(scale.to(torch.float16)[:, None]).clamp_(-E4M3_MAX, E4M3_MAX).to(_T[kind])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    s = {"case": case}
    op, dt = case["op"], _T[case["dtype"]]
    if op == "norm":
        # a residual stream: a few channels far larger than the rest
        gain = torch.where(torch.rand(case["n"], generator=g, device="cuda") < 0.01, 20.0, 1.0)
        s["x"] = rand(case["rows"], case["n"]).to(dt)
        if case["residual"]:
            s["residual"] = (rand(case["rows"], case["n"]) * gain * 2).to(dt)
        s["weight"] = (1 + 0.2 * rand(case["n"])).to(dt)
    elif op == "linear":
        m, n, k, groups = case["m"], case["n"], case["k"], case["k"] // case["group"]
        x = rand(m, k)
        if case["dtype"] == "e4m3":
            s["x_scale"] = x.abs().amax(1) / E4M3_MAX
            x = (x / s["x_scale"][:, None]).clamp(-E4M3_MAX, E4M3_MAX)
        s["x"] = x.to(dt)
        s["qweight"] = torch.randint(0, 256, (n, k // 2), generator=g, device="cuda",
                                     dtype=torch.uint8)
        u = torch.rand(groups, n, generator=g, device="cuda")
        s["scales"] = ((0.5 + u) / (4 * math.sqrt(k))).to(_T[case["out"]])
        s["zeros"] = torch.randint(4, 12, (groups, n), generator=g, device="cuda",
                                   dtype=torch.uint8) if case["zeros"] else None
        if own:
            from sketchpad_b200 import Int4Linear
            s["layer"] = Int4Linear(s["qweight"], s["scales"], s["zeros"],
                                    group_size=case["group"])
    else:
        hq, hkv, d, page, b = case["hq"], case["hkv"], case["d"], case["page"], case["seqs"]
        ks = vs = None
        if case["cache"] == "e4m3":
            ks = 0.01 + 0.01 * torch.rand(hkv, generator=g, device="cuda")
            vs = 0.01 + 0.01 * torch.rand(hkv, generator=g, device="cuda")
        if op == "append":
            ends = [case["start"] + case["chunk"] * (1 + i % 2) for i in range(b)]
            s["table"], total = _pages(ends, page, g)
            first = torch.tensor(ends, device="cuda") - case["chunk"]
            pos = first[:, None] + torch.arange(case["chunk"], device="cuda")
            s["positions"] = pos.reshape(-1).to(torch.int32)
            s["seq_ids"] = torch.arange(b, device="cuda").repeat_interleave(case["chunk"]).to(
                torch.int32)
            t = b * case["chunk"]
            # the three parts of one projection's output, each a view of its columns
            qkv = rand(t, hq + 2 * hkv, d).to(dt)
            s["q"], s["k"], s["v"] = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
            ang = torch.arange(max(ends), device="cuda")[:, None] * torch.exp(
                torch.arange(d // 2, device="cuda") * (-2 * math.log(10000.0) / d))
            s["rope"] = torch.stack((ang.cos(), ang.sin()), -1).float().contiguous()
        else:
            lens = _lengths(case)
            order = torch.randperm(b, generator=g, device="cuda").tolist()
            lens = [lens[i] for i in order]
            s["table"], total = _pages(lens, page, g)
            s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
            s["q"] = rand(b, hq, d).to(dt)
        s["k_cache"] = _cache_fill((total, page, hkv, d), case["cache"], ks, g)
        s["v_cache"] = _cache_fill((total, page, hkv, d), case["cache"], vs, g)
        s["k_scale"], s["v_scale"] = ks, vs
        if own:
            from sketchpad_b200 import PagedKVCache
            s["cache"] = PagedKVCache(s["k_cache"], s["v_cache"], ks, vs)
    return s


# ------------------------------------------------------------------------------- one pass
def run(s):
    return (_own if own else _plain)[s["case"]["op"]](s)


def _own_norm(s):
    from sketchpad_b200 import rms_norm, rms_norm_fp8
    f = rms_norm_fp8 if s["case"]["fp8"] else rms_norm
    return f(s["x"], s["weight"], EPS, residual=s.get("residual"))


def _own_linear(s):
    return s["layer"](s["x"], s.get("x_scale"), out_dtype=_T[s["case"]["out"]])


def _own_append(s):
    q = s["cache"].append(s["k"], s["v"], s["table"], s["seq_ids"], s["positions"], q=s["q"],
                          rope=s["rope"])
    return q, s["k_cache"], s["v_cache"]


def _own_attend(s):
    c = s["case"]
    return s["cache"].attend(s["q"], s["table"], s["lens"], window=c["window"] or None,
                             sinks=c["sinks"])


def _plain_norm(s):
    c, x = s["case"], s["x"].float()
    extra = ()
    if c["residual"]:
        extra = ((x + s["residual"].float()).to(s["x"].dtype),)
        x = extra[0].float()
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * s["weight"].float()
    if not c["fp8"]:
        return (y.to(s["x"].dtype),) + extra if extra else y.to(s["x"].dtype)
    amax = y.abs().amax(-1)
    scale = torch.where(amax == 0, 1.0, amax / E4M3_MAX)
    q = (y / scale[:, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    return (q, scale) + extra


def _weights(s, dtype):
    q = s["qweight"]
    w = torch.stack((q & 15, q >> 4), -1).reshape(q.shape[0], -1)
    w = w.reshape(q.shape[0], -1, s["case"]["group"]).to(dtype)
    z = 8.0 if s["zeros"] is None else s["zeros"].t()[:, :, None].to(dtype)
    return ((w - z) * s["scales"].t()[:, :, None].to(dtype)).reshape(q.shape[0], -1)


def _plain_linear(s):
    x = s["x"].float()
    if "x_scale" in s:
        x = x * s["x_scale"][:, None]
    return (x @ _weights(s, torch.float32).t()).to(_T[s["case"]["out"]])


def _rotate(x, cs):
    c, n = cs[:, None, :, 0], cs[:, None, :, 1]
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack((a * c - b * n, b * c + a * n), -1).reshape(x.shape)


def _store(cache, page, slot, new, scale):
    if scale is None:
        cache[page, slot] = new.to(cache.dtype)
    else:
        new = (new / scale[:, None]).clamp(-E4M3_MAX, E4M3_MAX).to(cache.dtype)
        cache.view(torch.uint8)[page, slot] = new.view(torch.uint8)


def _plain_append(s):
    pos, page = s["positions"].long(), s["case"]["page"]
    at = s["table"][s["seq_ids"].long(), pos // page].long()
    cs = s["rope"][pos]
    _store(s["k_cache"], at, pos % page, _rotate(s["k"].float(), cs), s["k_scale"])
    _store(s["v_cache"], at, pos % page, s["v"].float(), s["v_scale"])
    return _rotate(s["q"].float(), cs).to(s["q"].dtype), s["k_cache"], s["v_cache"]


def _gather(cache, at, slot, scale):
    v = (cache.view(torch.uint8)[at, slot].view(cache.dtype) if scale is not None
         else cache[at, slot]).float()
    return v if scale is None else v * scale[:, None]


def _plain_attend(s):
    c = s["case"]
    b, hq, d = s["q"].shape
    pos = torch.arange(s["table"].shape[1] * c["page"], device="cuda")
    n = s["lens"][:, None].long()
    seen = pos < n
    if c["window"]:
        seen = seen & ((pos >= n - c["window"]) | (pos < c["sinks"]))
    at = s["table"].long().clamp(min=0)[:, pos // c["page"]]
    slot = (pos % c["page"]).expand(b, -1)
    k = _gather(s["k_cache"], at, slot, s["k_scale"]).permute(0, 2, 3, 1)  # [b, hkv, d, L]
    q = s["q"].float().reshape(b, c["hkv"], -1, d)
    sc = (torch.matmul(q, k) / math.sqrt(d)).masked_fill(~seen[:, None, None], float("-inf"))
    m = sc.amax(-1, keepdim=True)
    p = torch.exp(sc - torch.where(m == float("-inf"), 0.0, m))
    v = _gather(s["v_cache"], at, slot, s["v_scale"])
    o = torch.matmul(p / p.sum(-1, keepdim=True).clamp(min=1e-30), v.permute(0, 2, 1, 3))
    return o.reshape(b, hq, d).to(s["q"].dtype)


_own = {"norm": _own_norm, "linear": _own_linear, "append": _own_append, "attend": _own_attend}
_plain = {"norm": _plain_norm, "linear": _plain_linear, "append": _plain_append,
          "attend": _plain_attend}


# ------------------------------------------------------------------------------- exact values
def exact(case, seed):
    """The operators' definitions in 64 bits, a sequence or a block of outputs at a time."""
    s = prepare(case, seed)
    f64 = torch.float64
    if case["op"] == "norm":
        x, extra = s["x"].to(f64), ()
        if case["residual"]:
            total = x + s["residual"].to(f64)
            x, extra = total.to(s["x"].dtype).to(f64), (total,)
        y = x / (x.pow(2).sum(-1, keepdim=True) / case["n"] + EPS).sqrt() * s["weight"].to(f64)
        if not case["fp8"]:
            return (y,) + extra if extra else y
        scale = y.abs().max(-1).values / E4M3_MAX
        scale[scale == 0] = 1
        return (y / scale[:, None], scale) + extra
    if case["op"] == "linear":
        x, parts = s["x"].to(f64), []
        if case["dtype"] == "e4m3":
            x = x * s["x_scale"].to(f64)[:, None]
        for lo in range(0, case["n"], 4096):
            q = s["qweight"][lo:lo + 4096]
            w = torch.empty(q.shape[0], case["k"], dtype=f64, device="cuda")
            w[:, 0::2], w[:, 1::2] = (q % 16).to(f64), (q // 16).to(f64)
            z = s["zeros"][:, lo:lo + 4096].to(f64).t() if case["zeros"] else torch.full(
                (q.shape[0], case["k"] // case["group"]), 8.0, dtype=f64, device="cuda")
            w -= z.repeat_interleave(case["group"], 1)
            w *= s["scales"][:, lo:lo + 4096].to(f64).t().repeat_interleave(case["group"], 1)
            parts.append(x @ w.t())
        return torch.cat(parts, 1)
    if case["op"] == "append":
        pos, page, d = s["positions"].long(), case["page"], case["d"]
        z = torch.view_as_complex(s["rope"].to(f64))[pos][:, None]
        turn = lambda t: torch.view_as_real(torch.view_as_complex(  # noqa: E731
            t.to(f64).reshape(*t.shape[:2], d // 2, 2).contiguous()) * z).reshape(t.shape)
        flat = s["table"][s["seq_ids"].long(), pos // page].long() * page + pos % page
        out = []
        for name, new in (("k", turn(s["k"])), ("v", s["v"].to(f64))):
            cache = s[name + "_cache"].to(f64)
            if case["cache"] == "e4m3":
                new = new / s[name + "_scale"].to(f64)[:, None]
                new = new.clamp(-E4M3_MAX, E4M3_MAX)
            cache.reshape(-1, case["hkv"], d).index_copy_(0, flat, new)
            out.append(cache)
        return turn(s["q"]), out[0], out[1]
    out = torch.zeros(s["q"].shape, dtype=f64, device="cuda")
    hkv, d = case["hkv"], case["d"]
    for i, n in enumerate(s["lens"].tolist()):
        w = case["window"]
        pos = torch.arange(n, device="cuda")
        if w and n > w:
            pos = torch.cat((pos[:min(case["sinks"], n - w)], pos[n - w:]))
        flat = s["table"][i].long()[pos // case["page"]] * case["page"] + pos % case["page"]
        k = s["k_cache"].view(torch.uint8).reshape(-1, hkv, d * _SIZE[case["cache"]])[flat]
        v = s["v_cache"].view(torch.uint8).reshape(-1, hkv, d * _SIZE[case["cache"]])[flat]
        k, v = (t.view(_T[case["cache"]]).to(f64).transpose(0, 1) for t in (k, v))
        if case["cache"] == "e4m3":
            k, v = (t * z.to(f64)[:, None, None] for t, z in ((k, s["k_scale"]),
                                                              (v, s["v_scale"])))
        q = s["q"][i].to(f64).reshape(hkv, -1, d)
        p = torch.softmax(torch.bmm(q, k.transpose(1, 2)) / math.sqrt(d), -1)
        out[i] = torch.bmm(p, v).reshape(-1, d)
    return out
