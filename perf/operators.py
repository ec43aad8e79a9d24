"""The operators of the cache held in 4 bits: appending keys and values to its pages, with the rotary positions applied on
the way, and attention that reads it, for single tokens and for portions of prompts.

The cache. Of a token's key (value) of one kv head, D numbers x, are kept: a scale s = bf16(max x / 15 - min x / 15), a minimum
m = bf16(min x), and per number a code n = round((x - m) / s), ties to even, held to 0 .. 15 (0 where s is 0), all in 32 bits (a
fifteenth: times the 32-bit number next to 1/15). A code stands for m + s n. Keys are quantised as rotated: x_i cos t - x_(i + D/2) sin t and x_(i + D/2) cos t + x_i sin t, rounded to 32 bits, with the
angle t = position * frequency_i in 32 bits (as everywhere in this package).

One layer's cache is uint8 [pages, kv heads, page size, W], W = 32 C + 8, C = ceil(D / 32) chunks of 32 numbers. Eight
tokens of a page and kv head lie together: codes of the keys [C][8 tokens][16 bytes], of the values [C][8 tokens][16 bytes] (byte b of a
chunk: number 2b in the low four bits, 2b + 1 in the high ones; what D leaves of the last chunk is 0), then bfloat16 [8 tokens][s of the
key, m of the key, s of the value, m of the value].

Attention. Row r of request s at position p sees the keys j of that request with p - window < j <= p (window 0: all up to p):
    out_r = sum_j softmax_j(scale q_r . K_j) V_j,   0 where a row sees nothing (position -1: a padding row).
"""
import math

import torch

own = False

FIFTEENTH = 0.06666667014360428         # the 32-bit number next to 1/15

# heads, kv heads, head size: the sizes of bench.py's models (1B, 3B, 8B), of the tests' small ones, and of other layouts
# (one kv head for all, as many kv heads as heads, head sizes that are no power of two)
LAYOUTS = {"1b": (32, 8, 64), "3b": (24, 8, 128), "8b": (32, 8, 128), "small": (6, 3, 48), "one": (20, 1, 80), "all": (8, 8, 96),
           "wide": (8, 2, 256)}


def listed():
    def append(name, layout, dtype, tokens, page, start):
        return dict(name=name, op="append", layout=layout, dtype=dtype, tokens=tokens, page=page, start=start)

    def decode(name, layout, dtype, seqs, lo, hi, page=16, window=0, idle=0):
        return dict(name=name, op="decode", layout=layout, dtype=dtype, seqs=seqs, lo=lo, hi=hi, page=page, window=window, idle=idle)

    def portion(name, layout, dtype, seqs, new_lo, new_hi, ctx_lo, ctx_hi, page=16, window=0):
        return dict(name=name, op="portion", layout=layout, dtype=dtype, seqs=seqs, new_lo=new_lo, new_hi=new_hi, ctx_lo=ctx_lo,
                    ctx_hi=ctx_hi, page=page, window=window)
    return [
        # a decode step of 8 requests: one token each, all latency
        append("append 8", "1b", "bfloat16", 8, 16, 2200),
        # a full portion of a prompt far into a document
        append("append 2048", "8b", "bfloat16", 2048, 16, 120001),
        # the 32-bit engine, an odd portion, a head size and a page size that are no powers of two
        append("append f32 517", "small", "float32", 517, 24, 300),
        # one user early in a chat: the smallest call
        decode("decode 1x100", "1b", "bfloat16", 1, 100, 100),
        # a handful of chats at once
        decode("decode 8x2200", "1b", "bfloat16", 8, 2200, 2200),
        # a full batch of long requests: the cache is what a step reads
        decode("decode 64x8192", "8b", "bfloat16", 64, 8192, 8192),
        # one request over a very long document
        decode("decode 1x131072", "1b", "bfloat16", 1, 131072, 131072),
        # requests of very different lengths with padding rows behind them, three heads per kv head
        decode("decode ragged 40", "3b", "bfloat16", 40, 17, 4000, page=32, idle=3),
        # the 32-bit engine decoding a few requests
        decode("decode f32 6", "1b", "float32", 6, 90, 1501),
        # the first portion of a prompt: time to the first token
        portion("portion 2048", "1b", "bfloat16", 1, 2048, 2048, 0, 0),
        # a later portion of a long prompt at 8B
        portion("portion 2048 at 8192", "8b", "bfloat16", 1, 2048, 2048, 8192, 8192),
        # portions of several requests at once, of odd lengths, in a window
        portion("portions ragged 5", "3b", "bfloat16", 5, 33, 700, 0, 1501, window=1024),
    ]


def _spread(n, lo, hi):
    """n whole numbers between lo and hi, evenly spread in logarithm, in an order that is no order."""
    if n == 1:
        return [hi]
    got = [int(round((lo + 1) * ((hi + 1) / (lo + 1)) ** (i / (n - 1)))) - 1 for i in range(n)]
    step = next(s for s in (7, 5, 3, 2, 1) if math.gcd(s, n) == 1)
    return [got[(i * step + n // 2) % n] for i in range(n)]


def _lens(case):
    """(cached before the call, new) tokens of every request."""
    if case["op"] == "decode":
        return [(n - 1, 1) for n in _spread(case["seqs"], case["lo"], case["hi"])]
    return list(zip(_spread(case["seqs"], case["ctx_lo"], case["ctx_hi"]), _spread(case["seqs"], case["new_lo"], case["new_hi"])[::-1]))


def _pairs(case):
    """(row, key) pairs that attention looks at, and distinct keys that it has to read."""
    w, pairs, keys = case["window"], 0, 0
    for ctx, new in _lens(case):
        if w:
            full = max(0, min(new, w - ctx))            # rows that see every earlier key
            pairs += full * ctx + full * (full + 1) // 2 + (new - full) * w
            keys += min(ctx + new, w + new - 1)
        else:
            pairs += new * ctx + new * (new + 1) // 2
            keys += ctx + new
    return pairs, keys


def _width(hd):
    return 32 * -(-hd // 32) + 8


def work(case):
    H, G, D = LAYOUTS[case["layout"]]
    es = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "append":
        # q, k, v in; q, the cache's bytes and the values that it now holds out
        T = case["tokens"]
        return {"bytes": T * (2 * H * D * es + 4 * G * D * es + G * _width(D)), "flops": T * (3 * (H + G) * D + 10 * G * D)}
    pairs, keys = _pairs(case)
    rows = sum(n for _, n in _lens(case))
    return {"bytes": keys * G * _width(D) + 2 * rows * H * D * es, "flops": 4 * pairs * H * D}


def _cost(case):
    w = work(case)
    return w["bytes"] / 6e12 + w["flops"] / (2e13 if case["dtype"] == "float32" else 1e15)


def draw(rng):
    most = max(_cost(c) for c in listed())
    sizes = {n: max(LAYOUTS[n][0] * LAYOUTS[n][2], 1) for n in LAYOUTS}

    def spread(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))
    while True:
        op = rng.choice(("append", "decode", "decode", "portion", "portion"))
        layout = rng.choice(("1b", "1b", "3b", "8b", "8b", "small", "one", "all", "wide"))
        dtype = rng.choice(("bfloat16", "bfloat16", "bfloat16", "float32"))
        page = rng.choice((8, 16, 16, 24, 32, 64))
        window = rng.choice((0, 0, spread(1, 2048)))
        f32 = dtype == "float32"
        if op == "append":
            case = dict(op=op, layout=layout, dtype=dtype, tokens=spread(1, 4096), page=page, start=spread(1, 130000))
        elif op == "decode":
            n = spread(1, 16 if f32 else 128)
            lo, hi = sorted((spread(1, 4096 if f32 else 65536), spread(1, 4096 if f32 else 65536)))
            case = dict(op=op, layout=layout, dtype=dtype, seqs=n, lo=hi if n == 1 else lo, hi=hi, page=page, window=window,
                        idle=rng.choice((0, 0, 1, 5)))
        else:
            n = spread(1, 4 if f32 else 12)
            a, b = sorted((spread(1, 600 if f32 else 2048), spread(1, 600 if f32 else 2048)))
            c, d = sorted((rng.choice((0, spread(1, 1000 if f32 else 8192))), rng.choice((0, spread(1, 1000 if f32 else 8192)))))
            if n == 1:
                a, c = b, d
            case = dict(op=op, layout=layout, dtype=dtype, seqs=n, new_lo=a, new_hi=b, ctx_lo=c, ctx_hi=d, page=page, window=window)
        if op == "append":
            if _cost(case) <= most:
                return case
            continue
        # the plain form works on rows and keys padded to the longest: what it holds stays bounded
        longest = max(c + n for c, n in _lens(case))
        new = max(n for _, n in _lens(case))
        held = case["seqs"] * longest * (2 * LAYOUTS[layout][1] * LAYOUTS[layout][2] + new * LAYOUTS[layout][0])
        if _cost(case) <= most and held <= 1.1e9 and sizes[layout]:
            return case


# ------------------------------------------------------------------------------------------------ what a program has in hand
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) + 12345)
    return g


def _quantise(x):
    """x float32 [..., D] -> (codes uint8 [..., D], scale, minimum bfloat16 [...])."""
    lo, hi = x.amin(-1), x.amax(-1)
    m = lo.to(torch.bfloat16)
    s = (hi * FIFTEENTH - lo * FIFTEENTH).to(torch.bfloat16)
    n = torch.round((x - m.float()[..., None]) / s.float()[..., None]).clamp_(0.0, 15.0)
    n = torch.where((s == 0)[..., None], torch.zeros_like(n), n)
    return n.to(torch.uint8), s, m


def _pack_codes(n, hd):
    """codes [N, 8 tokens, D] -> bytes [N, C * 8 * 16] as the cache holds them."""
    C = -(-hd // 32)
    if 32 * C != hd:
        n = torch.nn.functional.pad(n, (0, 32 * C - hd))
    b = n[..., 0::2] | (n[..., 1::2] << 4)
    return b.view(n.shape[0], 8, C, 16).transpose(1, 2).reshape(n.shape[0], C * 128)


def _tiles(k, v, hd):
    """keys and values float32 [N, 8, D] -> the bytes of N groups of eight tokens [N, 8 W]."""
    (kn, ks, km), (vn, vs, vm) = _quantise(k), _quantise(v)
    par = torch.stack((ks, km, vs, vm), dim=-1).contiguous().view(torch.uint8).reshape(k.shape[0], 64)
    return torch.cat((_pack_codes(kn, hd), _pack_codes(vn, hd), par), dim=1)


def _unpack(cache, hd):
    """cache [pages, G, P, W] -> keys and values float32 [pages, G, P, D] that its codes stand for."""
    pages, G, P, W = cache.shape
    C = -(-hd // 32)
    t = cache.view(pages * G * (P // 8), 8 * W)
    par = t[:, 256 * C:].reshape(-1, 8, 8).view(torch.bfloat16).float()
    got = []
    for i in (0, 1):
        b = t[:, 128 * C * i:128 * C * (i + 1)].reshape(-1, C, 8, 16).transpose(1, 2)
        n = torch.stack((b & 15, b >> 4), dim=-1).reshape(-1, 8, 32 * C)[..., :hd].float()
        n *= par[..., 2 * i, None]
        n += par[..., 2 * i + 1, None]
        got.append(n.view(pages, G, P, hd))
    return got


def _inv_freq(hd):
    return torch.tensor([500000.0 ** (-2.0 * i / hd) for i in range(hd // 2)], dtype=torch.float32, device="cuda")


def prepare(case, seed):
    H, G, D = LAYOUTS[case["layout"]]
    dt = getattr(torch, case["dtype"])
    g = _generator(seed)
    P, W = case["page"], _width(D)
    i32 = dict(dtype=torch.int32, device="cuda")

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")
    # a few features of the keys stand out in every token, as in trained models; some tokens' values are larger than others'
    gain = 1.0 + 3.0 * (torch.rand(G, D, generator=g, device="cuda") < 0.05)
    if case["op"] == "append":
        T = case["tokens"]
        # the projection's output [q | k | v], one row per token
        qkv = torch.cat((1.5 * normal(T, H * D), (normal(T, G, D) * gain).reshape(T, G * D), normal(T, G * D)), dim=1).to(dt)
        pages = -(-T // P) + 3
        order = torch.randperm(pages, generator=g, device="cuda")
        at = torch.arange(T, device="cuda") + 5              # the portion starts inside a page
        slots = (order[at // P] * P + at % P).to(torch.int32)
        if T <= 64:                                          # a decode step: every token in a page of its own request
            slots = (torch.randperm(T + 3, generator=g, device="cuda")[:T] * P + torch.arange(T, device="cuda") * 5 % P).to(torch.int32)
            pages = T + 3
        positions = (torch.arange(T, device="cuda") + case["start"]).to(torch.int32)
        return dict(op="append", sizes=(H, G, D), qkv=qkv, positions=positions, slots=slots, inv_freq=_inv_freq(D),
                    cache=torch.zeros((pages, G, P, W), dtype=torch.uint8, device="cuda"),
                    q_out=torch.empty((T, H * D), dtype=dt, device="cuda"),
                    k_out=torch.empty((T, G * D), dtype=dt, device="cuda"), v_out=torch.empty((T, G * D), dtype=dt, device="cuda"))
    lens = _lens(case)
    S, idle = len(lens), case.get("idle", 0)
    need = [-(-(c + n) // P) for c, n in lens]
    total, most = sum(need) + 2, max(need)
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    tables, at = torch.zeros((S + idle, most), **i32), 0
    for s, n in enumerate(need):
        tables[s, :n] = order[at:at + n]
        at += n
    cache = torch.empty((total * G * (P // 8), 8 * W), dtype=torch.uint8, device="cuda")
    groups = cache.shape[0]
    head = torch.arange(groups, device="cuda") // (P // 8) % G
    for a in range(0, groups, 1 << 19):
        n = min(1 << 19, groups - a)
        cache[a:a + n] = _tiles(normal(n, 8, D) * gain[head[a:a + n], None], normal(n, 8, D) * (0.5 + torch.rand(n, 8, 1, generator=g, device="cuda")), D)
    rows = sum(n for _, n in lens) + idle
    q = normal(rows, H * D).to(dt)
    out = torch.empty_like(q)
    starts, pos, seq = [0], [], []
    for s, (c, n) in enumerate(lens):
        starts.append(starts[-1] + n)
        pos += range(c, c + n)
        seq += [s] * n
    pos += [-1] * idle
    state = dict(op=case["op"], sizes=(H, G, D), scale=1.0 / math.sqrt(D), window=case["window"], q=q, out=out,
                 cache=cache.view(total, G, P, W), tables=tables, positions=torch.tensor(pos, **i32), seqs=S, new=max(n for _, n in lens),
                 starts=torch.tensor(starts, **i32), contexts=torch.tensor([c for c, _ in lens], **i32),
                 row_seq=torch.tensor(seq + list(range(S, S + idle)), **i32).long(), scratch=None)
    if own and case["op"] == "decode":
        from vllm_oxide_b200 import kernels
        state["scratch"] = kernels.kv4_scratch(S + idle, H, G, D, "cuda")
    return state


# ------------------------------------------------------------------------------------------------ the operators
def _append(st):
    H, G, D = st["sizes"]
    q, k, v = st["qkv"].split((H * D, G * D, G * D), dim=1)
    if own:
        from vllm_oxide_b200 import kernels
        kernels.kv4_append(q, k, v, st["positions"], st["slots"], st["inv_freq"], st["cache"], H, G, D, q_out=st["q_out"])
        kernels.kv4_read(st["cache"], st["slots"], st["k_out"], st["v_out"], G, D)
        return {"q": st["q_out"], "k": st["k_out"], "v": st["v_out"]}
    T, dt = q.shape[0], q.dtype
    # the rotation in 64 bits: a key next to the border of two codes falls to the right side
    t = (st["positions"].float()[:, None] * st["inv_freq"]).double()
    c, s = t.cos()[:, None], t.sin()[:, None]

    def rotate(x):
        a, b = x.double().split(D // 2, dim=-1)
        return torch.cat((a * c - b * s, b * c + a * s), dim=-1)
    k32 = rotate(k.reshape(T, G, D)).float()
    v32 = v.reshape(T, G, D).float()
    # eight tokens of a page lie together: the codes of a token go to its bytes of each chunk
    cache = st["cache"]
    pages, _, P, W = cache.shape
    C = -(-D // 32)
    one = _tiles(k32.reshape(T * G, 1, D).expand(-1, 8, -1), v32.reshape(T * G, 1, D).expand(-1, 8, -1), D)
    slot = st["slots"].long()
    group = ((slot // P)[:, None] * G + torch.arange(G, device=q.device)) * (P // 8) + (slot % P // 8)[:, None]
    lane = (slot % 8)[:, None].expand(T, G).reshape(-1)
    byte = torch.arange(16, device=q.device)
    # its bytes inside the group: 2 C chunks of 16 bytes, 128 apart, and 8 bytes of scales and minima
    at = torch.cat(((torch.arange(2 * C, device=q.device) * 128)[:, None].add(byte).reshape(1, -1) + 16 * lane[:, None],
                    256 * C + 8 * lane[:, None] + byte[:8]), dim=1)
    tiles = cache.view(-1, 8 * W)
    tiles[group.reshape(-1, 1), at] = one.gather(1, at)
    keys, values = _unpack(tiles[group.reshape(-1)].view(T * G, 1, 8, W), D)
    pick = torch.arange(T * G, device=q.device)
    return {"q": rotate(q.reshape(T, H, D)).to(dt).view(T, H * D), "k": keys[pick, 0, lane].to(dt).view(T, G * D),
            "v": values[pick, 0, lane].to(dt).view(T, G * D)}


def _attend(st):
    H, G, D = st["sizes"]
    q, out = st["q"], st["out"]
    if own:
        from vllm_oxide_b200 import kernels
        if st["op"] == "decode":
            kernels.attn_decode_kv4(q, out, st["cache"], st["tables"], st["positions"], H, G, D, st["scale"], window=st["window"],
                                    scratch=st["scratch"])
        else:
            kernels.attn_prefill_kv4(q, out, st["cache"], st["tables"], st["starts"], st["contexts"], st["seqs"], st["new"], H, G, D,
                                     st["scale"], window=st["window"])
        return out
    rows, P = q.shape[0], st["cache"].shape[2]
    tables = st["tables"].long()
    S, L = tables.shape[0], tables.shape[1] * P
    # every request's pages side by side, rows padded to the longest portion of a request
    keys, values = (x.transpose(1, 2).reshape(S, L, G, D) for x in _unpack(st["cache"][tables.reshape(-1)], D))
    first = torch.cat((st["starts"][:-1], torch.arange(S - st["seqs"], device=q.device, dtype=torch.int32) + rows - (S - st["seqs"]))).long()
    row = torch.arange(rows, device=q.device) - first[st["row_seq"]]
    qs = torch.zeros((S, st["new"], G, H // G, D), device=q.device)
    qs[st["row_seq"], row] = q.float().view(rows, G, H // G, D) * st["scale"]
    pos = torch.full((S, st["new"]), -1, device=q.device, dtype=torch.int32)
    pos[st["row_seq"], row] = st["positions"]
    j = torch.arange(L, device=q.device)
    seen = (j <= pos[..., None]) if not st["window"] else (j <= pos[..., None]) & (j > pos[..., None] - st["window"])
    score = torch.einsum("snghd,slgd->sgnhl", qs, keys)
    seen = seen[:, None, :, None]
    score = score.masked_fill_(~seen, -math.inf)
    p = torch.exp(score.sub_(score.amax(-1, keepdim=True).clamp_min(-1e30)))
    o = torch.einsum("sgnhl,slgd->snghd", p, values) / p.sum(-1).clamp_min(1e-30).permute(0, 2, 1, 3)[..., None]
    return o.reshape(S, st["new"], H * D)[st["row_seq"], row].to(q.dtype)


def run(state):
    return _append(state) if state["op"] == "append" else _attend(state)


# ------------------------------------------------------------------------------------------------ 64 bits
def _exact_codes(x):
    """x float32 [..., D] -> what the cache makes of them, float64. The steps that the definition takes in 32 bits are taken so."""
    low, high = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values
    m = low.bfloat16().float()
    s = (high * FIFTEENTH - low * FIFTEENTH).bfloat16().float()
    n = torch.where(s > 0, (x - m) / torch.where(s > 0, s, 1.0), 0.0).double()
    odd_tie = (n % 1 == 0.5) & (torch.floor(n) % 2 == 0)
    return m.double() + s.double() * (torch.floor(n + 0.5) - odd_tie.double()).clamp(0, 15)


def _exact_values(cache, page, head, offset, hd):
    """Key and value float64 [..., D] of the tokens at (page, head, offset), byte by byte."""
    P, W = cache.shape[2:]
    C = (hd + 31) // 32
    flat = cache.reshape(-1)
    base = ((page * cache.shape[1] + head) * P + offset // 8 * 8) * W
    t = offset % 8
    d = torch.arange(hd, device=cache.device)
    out = []
    for which in (0, 1):
        at = (base + 16 * t)[..., None] + (which * C + d // 32) * 128 + d % 32 // 2
        n = flat[at].int() >> (4 * (d % 2)).int() & 15
        pos = base + 256 * C + 8 * t + 4 * which
        two = [(flat[pos + 2 * i + 1].int() << 24 | flat[pos + 2 * i].int() << 16).view(torch.float32).double() for i in (0, 1)]
        out.append(two[1][..., None] + two[0][..., None] * n)
    return out


def exact(case, seed):
    st = prepare(case, seed)
    H, G, D = st["sizes"]
    if case["op"] == "append":
        T = case["tokens"]
        x = st["qkv"].double().view(T, H + 2 * G, D)
        angle = (st["positions"].float()[:, None] * st["inv_freq"][None]).double()[:, None]
        turn = torch.polar(torch.ones_like(angle), angle)
        z = torch.complex(x[..., :D // 2], x[..., D // 2:])[:, :H + G] * turn
        x = torch.cat((torch.cat((z.real, z.imag), dim=-1), x[:, H + G:]), dim=1)
        kv = _exact_codes(x[:, H:].float()).view(T, 2, G * D)
        return {"q": x[:, :H].reshape(T, H * D), "k": kv[:, 0], "v": kv[:, 1]}
    out = torch.zeros((st["q"].shape[0], H * D), dtype=torch.float64, device="cuda")
    P, w, at = case["page"], case["window"], 0
    heads = torch.arange(G, device="cuda")[:, None]
    for s, (ctx, new) in enumerate(_lens(case)):
        total = ctx + new
        lo = max(0, ctx + 1 - w) if w else 0
        j = torch.arange(lo, total, device="cuda")
        k, v = _exact_values(st["cache"], st["tables"][s].long()[j // P], heads, j % P, D)       # [G, keys, D]
        for a in range(0, new, 256):
            b = min(new, a + 256)
            q = st["q"][at + a:at + b].double().view(b - a, G, H // G, D).permute(1, 2, 0, 3).reshape(G, -1, D)
            x = (q @ k.transpose(1, 2)).view(G, H // G, b - a, -1) * st["scale"]
            p = torch.arange(ctx + a, ctx + b, device="cuda")[:, None]
            x = x.masked_fill((j > p) | ((j <= p - w) if w else False), -math.inf)
            o = torch.softmax(x, -1).view(G, -1, total - lo) @ v
            out[at + a:at + b] = o.view(G, H // G, b - a, D).permute(2, 0, 1, 3).reshape(b - a, H * D)
        at += new
    return out
