"""What is measured of the 4-bit key / value cache: writing it, reading it back and attending over it.

The cache of one layer is a pair of tensors (two pairs for keys and values, one for a latent cache that
is both):

    codes   uint8 [B, Hk, L, W / 2]     byte i of a row holds dims 2i (low nibble) and 2i + 1
    params  bf16  [B, Hk, L, W / g, 2]  (scale s, smallest value m) of each group of g = 64 dims

and stands for x = n * s + m with n = 0 .. 15.  A group is written as m = bf16(min x),
s = bf16((max x - m) / 15) (that quotient in fp32) and n = clamp(round((x - m) / s), 0, 15).
Position p of a sequence lies in row `sink + p`; rows [0, n_sink) hold compressed memory that every
query sees.  A query at position t sees the positions p < kv_len, p <= t and, with a window, p > t - window.
"""
import math

import torch

own = False

GROUP = 64
_DEV = "cuda"


# ----------------------------------------------------------------------------------------------
# cases
# ----------------------------------------------------------------------------------------------
def listed():
    return [
        # --- attention over a key / value cache with grouped heads -------------------------------
        # first tokens of a chat answered by the draft model: latency of the call is all there is
        _attend("draft_b1_short", B=1, H=8, Hk=8, D=128, ctx=130),
        # one long conversation on the dense model
        _attend("dense_b1_long", B=1, H=48, Hk=8, D=128, ctx=8192),
        # the serving batch of the long-context benchmark on the dense model's heads
        _attend("dense_b64_long", B=64, H=48, Hk=8, D=128, ctx=8192),
        # verifying four drafted tokens, sequences of uneven length, a window and memory rows
        _attend("verify_b16_window", B=16, H=8, Hk=8, D=128, ctx=4001, Tn=5, ragged=True, window=1024, sink=64),
        # heads of 64, an odd batch, short uneven sequences
        _attend("small_heads_b7", B=7, H=16, Hk=2, D=64, ctx=1500, ragged=True),
        # --- attention over a latent cache --------------------------------------------------------
        # one long conversation on the latent-attention model
        _attend("latent_b1_long", B=1, H=16, rank=512, rope=64, ctx=8192),
        # the long-context serving benchmark: window of 4096 and 64 memory rows
        _attend("latent_b64_window", B=64, H=16, rank=512, rope=64, ctx=8192, window=4096, sink=64),
        # verifying three drafted tokens on the smaller latent
        _attend("latent_verify_b8", B=8, H=16, rank=256, rope=64, ctx=4099, Tn=4, ragged=True),
        # --- writing the cache and reading it back ------------------------------------------------
        # the new token of every sequence of the serving batch (keys and values)
        _store("append_dense_b64", B=64, Hk=8, W=128, T=1, ctx=2048),
        # the same for a latent cache
        _store("append_latent_b64", B=64, Hk=1, W=576, T=1, ctx=2048, pair=False),
        # prompts of uneven batch and odd length entering the cache
        _store("prompt_dense_b3", B=3, Hk=8, W=128, T=4001, ctx=4096),
        # long prompts of the latent-attention model
        _store("prompt_latent_b8", B=8, Hk=1, W=576, T=8192, ctx=8192, pair=False),
    ]


def _attend(name, B, H, ctx, Hk=1, D=0, rank=0, rope=0, Tn=1, ragged=False, window=0, sink=0):
    return {"name": name, "op": "attend", "B": B, "H": H, "Hk": Hk, "D": D, "rank": rank, "rope": rope, "ctx": ctx,
            "Tn": Tn, "ragged": ragged, "window": window, "sink": sink}


def _store(name, B, Hk, W, T, ctx, pair=True):
    return {"name": name, "op": "store", "B": B, "Hk": Hk, "W": W, "T": T, "ctx": ctx, "pair": pair}


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["heads", "heads", "latent", "latent", "store"])
    B = _log_int(rng, 1, 64)
    if kind == "store":
        pair = rng.random() < 0.5
        T = 1 if rng.random() < 0.3 else min(_log_int(rng, 2, 8192), 65536 // B)
        Hk, W = (rng.choice([(8, 128), (2, 64), (4, 128)]) if pair else rng.choice([(1, 576), (1, 320)]))
        c = _store("", B, Hk, W, T, T + rng.randint(0, 300), pair)
    else:
        Tn = 1 if rng.random() < 0.6 else rng.randint(2, 6)
        ctx = max(Tn, _log_int(rng, 1, 8192))
        kw = {"B": B, "ctx": ctx, "Tn": Tn, "ragged": rng.random() < 0.5,
              "window": rng.choice([0, 0, rng.randint(1, 4096)]), "sink": rng.choice([0, 0, rng.randint(1, 64)])}
        if kind == "heads":
            H, Hk, D = rng.choice([(48, 8, 128), (8, 8, 128), (16, 2, 64), (16, 4, 128)])
            c = _attend("", H=H, Hk=Hk, D=D, **kw)
        else:
            c = _attend("", H=16, rank=rng.choice([512, 256]), rope=64, **kw)
    del c["name"]
    return c


# ----------------------------------------------------------------------------------------------
# sizes that follow from a case
# ----------------------------------------------------------------------------------------------
def _round_up(n, m):
    return (n + m - 1) // m * m


def _lengths(c):
    """Cached positions of each sequence, the new ones included."""
    B, ctx, Tn = c["B"], c["ctx"], c["Tn"]
    if not c["ragged"]:
        return [ctx] * B
    lo = max(Tn, ctx // 4)
    return [lo + int((ctx - lo) * ((0.618034 * (b + 1)) % 1.0)) for b in range(B)]


def _visible(c):
    """Cache rows that at least one query of each sequence sees, summed over the sequences."""
    total = 0
    for n in _lengths(c):
        first = max(0, n - c["Tn"] - c["window"] + 1) if c["window"] else 0
        total += n - first + c["sink"]
    return total


def work(case):
    c = case
    if c["op"] == "store":
        elems = c["B"] * c["T"] * c["Hk"] * c["W"] * (2 if c["pair"] else 1)
        # bf16 rows in, codes and parameters written, bf16 rows out
        return {"bytes": elems * (2 + 0.5 + 4 / GROUP + 2), "flops": elems * 6}
    rows = _visible(c)
    if c["rank"]:
        W, V = c["rank"] + c["rope"], c["rank"]
        cache = rows * (W // 2 + 4 * W // GROUP)
    else:
        W = V = c["D"]
        cache = rows * c["Hk"] * 2 * (W // 2 + 4 * W // GROUP)
    queries = c["B"] * c["Tn"] * c["H"]
    return {"bytes": cache + 2 * queries * (W + V), "flops": 2 * rows * c["Tn"] * c["H"] * (W + V)}


# ----------------------------------------------------------------------------------------------
# inputs
# ----------------------------------------------------------------------------------------------
def _fill(codes, params, gen, sink, ctx):
    """A cache as a prompt leaves it: channels of uneven size, tokens of uneven norm, quantised by the
    rule at the top of this file; rows behind the context are empty."""
    B, Hk, L, half = codes.shape
    W = 2 * half
    channel = torch.exp(0.7 * torch.randn(Hk, 1, W, generator=gen, device=_DEV))
    shift = 0.5 * torch.randn(Hk, 1, W, generator=gen, device=_DEV)
    n = sink + ctx
    for b in range(B):
        token = torch.exp(0.3 * torch.randn(1, n, 1, generator=gen, device=_DEV))
        x = (torch.randn(Hk, n, W, generator=gen, device=_DEV) * token + shift) * channel
        x = x.to(torch.bfloat16).float().view(Hk, n, W // GROUP, GROUP)
        m = x.amin(-1).to(torch.bfloat16)
        s = ((x.amax(-1) - m.float()) / 15.0).to(torch.bfloat16)
        q = torch.round((x - m.float()[..., None]) / s.float()[..., None]).clamp_(0, 15).to(torch.uint8)
        q = q.view(Hk, n, half, 2)
        codes[b, :, :n] = q[..., 0] | (q[..., 1] << 4)
        params[b, :, :n, :, 0] = s
        params[b, :, :n, :, 1] = m


def _empty_cache(B, Hk, L, W):
    return (torch.zeros(B, Hk, L, W // 2, dtype=torch.uint8, device=_DEV),
            torch.zeros(B, Hk, L, W // GROUP, 2, dtype=torch.bfloat16, device=_DEV))


def prepare(case, seed):
    c = case
    gen = torch.Generator(device=_DEV).manual_seed(seed)
    st = {"case": dict(c)}
    if c["op"] == "store":
        B, Hk, W, T = c["B"], c["Hk"], c["W"], c["T"]
        L = _round_up(c["ctx"], 32)
        for name in ("k", "v")[:2 if c["pair"] else 1]:
            channel = torch.exp(0.7 * torch.randn(Hk, W, generator=gen, device=_DEV))
            x = torch.empty(B, T, Hk, W, dtype=torch.bfloat16, device=_DEV)
            for b in range(B):
                x[b] = (torch.randn(T, Hk, W, generator=gen, device=_DEV) * channel).to(torch.bfloat16)
            st[name] = x
            st[name + "c"], st[name + "p"] = _empty_cache(B, Hk, L, W)
        # prompts start at the front of the cache; a single token lands behind each sequence's text
        if T > 1:
            start = torch.zeros(B, 1, dtype=torch.int64, device=_DEV)
        else:
            start = torch.randint(0, c["ctx"], (B, 1), generator=gen, device=_DEV)
        st["pos"] = start + torch.arange(T, device=_DEV)[None]
        return st
    B, Tn, H, sink = c["B"], c["Tn"], c["H"], c["sink"]
    W = c["rank"] + c["rope"] if c["rank"] else c["D"]
    L = _round_up(sink + c["ctx"], 32)
    st["kc"], st["kp"] = _empty_cache(B, c["Hk"], L, W)
    _fill(st["kc"], st["kp"], gen, sink, c["ctx"])
    st["vc"] = st["vp"] = None
    if not c["rank"]:
        st["vc"], st["vp"] = _empty_cache(B, c["Hk"], L, W)
        _fill(st["vc"], st["vp"], gen, sink, c["ctx"])
    # queries whose largest scores stand out of the rest by a few units
    st["q"] = torch.randn(B, Tn, H, W, generator=gen, device=_DEV).to(torch.bfloat16)
    st["kv_len"] = torch.tensor(_lengths(c), dtype=torch.int32, device=_DEV)
    st["q_pos"] = st["kv_len"].long()[:, None] - Tn + torch.arange(Tn, device=_DEV)[None]
    st["scale"] = 1.0 / math.sqrt(c["D"] or 192)
    return st


# ----------------------------------------------------------------------------------------------
# one pass
# ----------------------------------------------------------------------------------------------
def run(state):
    c = state["case"]
    if c["op"] == "store":
        return _run_store(state)
    return _run_attend(state)


def _run_store(st):
    pair = st["case"]["pair"]
    if own:
        from omnicoder.ops.kv4 import kv4_read, kv4_write
        kv = (st["vc"], st["vp"]) if pair else (None, None)
        kv4_write(st["pos"], st["k"], st["kc"], st["kp"], st["v"] if pair else None, *kv)
        return kv4_read(st["pos"], st["kc"], st["kp"], *kv)
    out = []
    for name in ("k", "v")[:2 if pair else 1]:
        _plain_write(st[name], st["pos"], st[name + "c"], st[name + "p"])
        out.append(_plain_read(st["pos"], st[name + "c"], st[name + "p"]))
    return tuple(out) if pair else out[0]


def _plain_write(x, pos, codes, params):
    B, T, Hk, W = x.shape
    g = x.double().view(B, T, Hk, W // GROUP, GROUP)      # 64 bits: values next to a border between codes
    m = g.amin(-1).to(torch.bfloat16)
    s = ((g.amax(-1).float() - m.float()) / 15.0).to(torch.bfloat16)
    q = torch.round((g - m.double()[..., None]) / s.double()[..., None]).clamp(0, 15)
    q = torch.where((s == 0)[..., None], torch.zeros_like(q), q).to(torch.uint8).view(B, T, Hk, W // 2, 2)
    b = torch.arange(B, device=x.device)[:, None].expand(B, T)
    codes[b, :, pos] = q[..., 0] | (q[..., 1] << 4)
    params[b, :, pos] = torch.stack([s, m], -1)


def _plain_values(codes, params):
    """fp32 values [..., W] of codes [..., W / 2] and params [..., W / g, 2]."""
    n = torch.stack([codes & 15, codes >> 4], -1).view(*params.shape[:-1], GROUP).float()
    x = n * params[..., 0:1].float() + params[..., 1:2].float()
    return x.view(*codes.shape[:-1], 2 * codes.shape[-1])


def _plain_read(pos, codes, params):
    B, T = pos.shape
    b = torch.arange(B, device=pos.device)[:, None].expand(B, T)
    return _plain_values(codes[b, :, pos], params[b, :, pos]).to(torch.bfloat16)


def _run_attend(st):
    c = st["case"]
    if own:
        from omnicoder.ops.decode import decode_attention
        return decode_attention(st["q"], st["kc"], st["vc"], st["q_pos"], st["kv_len"], window=c["window"],
                                scale=st["scale"], k_scale=st["kp"], v_scale=st["vp"], latent_v_dim=c["rank"],
                                sink_rows=c["sink"], n_sink=c["sink"])
    q = st["q"]
    B, Tn, H, W = q.shape
    Hk = c["Hk"]
    k = _plain_values(st["kc"], st["kp"])                                       # [B, Hk, L, W]
    v = k[..., :c["rank"]] if c["rank"] else _plain_values(st["vc"], st["vp"])
    qr = q.float().view(B, Tn, Hk, H // Hk, W).permute(0, 2, 1, 3, 4).reshape(B, Hk, -1, W)
    s = torch.matmul(qr, k.transpose(-1, -2)) * st["scale"]                     # [B, Hk, Tn * G, L]
    row = torch.arange(k.shape[2], device=q.device)
    p = row - c["sink"]
    t = st["q_pos"][:, :, None]
    seen = (p >= 0) & (p < st["kv_len"].long()[:, None, None]) & (p <= t)
    if c["window"]:
        seen = seen & (p > t - c["window"])
    seen = seen | (row < c["sink"])                                             # [B, Tn, L]
    seen = seen[:, None, :, None].expand(B, Hk, Tn, H // Hk, -1).reshape(s.shape)
    s = s.masked_fill(~seen, float("-inf"))
    e = torch.exp(s - s.amax(-1, keepdim=True))
    o = torch.matmul(e, v) / e.sum(-1, keepdim=True)
    return o.view(B, Hk, Tn, H // Hk, -1).permute(0, 2, 1, 3, 4).reshape(B, Tn, H, -1).to(q.dtype)


# ----------------------------------------------------------------------------------------------
# the definition in 64 bits
# ----------------------------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "store":
        out = tuple(_exact_store(st[n]) for n in ("k", "v")[:2 if case["pair"] else 1])
        return out if case["pair"] else out[0]
    return torch.stack([_exact_sequence(st, case, b) for b in range(case["B"])])


def _exact_store(x):
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for b in range(x.shape[0]):
        for i in range(0, x.shape[-1], GROUP):
            g = x[b, ..., i:i + GROUP].to(torch.float64)
            low, high = g.min(-1, keepdim=True).values, g.max(-1, keepdim=True).values
            step = ((high - low).to(torch.float32) / 15).to(torch.bfloat16).to(torch.float64)
            n = torch.where(step > 0, ((g - low) / step).round(), torch.zeros_like(g))
            out[b, ..., i:i + GROUP] = torch.clamp(n, 0, 15) * step + low
    return out


def _exact_rows(codes, params):
    half = codes.shape[-1]
    x = torch.empty(*codes.shape[:-1], 2 * half, dtype=torch.float64, device=codes.device)
    x[..., 0::2] = (codes % 16).double()
    x[..., 1::2] = torch.div(codes, 16, rounding_mode="floor").double()
    scale = params[..., 0].double().repeat_interleave(GROUP, -1)
    least = params[..., 1].double().repeat_interleave(GROUP, -1)
    return x * scale + least


def _exact_sequence(st, c, b):
    n, Tn, sink = int(st["kv_len"][b]), c["Tn"], c["sink"]
    G = c["H"] // c["Hk"]
    k = _exact_rows(st["kc"][b, :, :sink + n], st["kp"][b, :, :sink + n])       # [Hk, rows, W]
    v = k[..., :c["rank"]] if c["rank"] else _exact_rows(st["vc"][b, :, :sink + n], st["vp"][b, :, :sink + n])
    out = []
    for i in range(Tn):
        t = n - Tn + i
        first = max(0, t - c["window"] + 1) if c["window"] else 0
        rows = torch.cat([torch.arange(sink, device=k.device),
                          torch.arange(sink + first, sink + t + 1, device=k.device)])
        qi = st["q"][b, i].double().view(c["Hk"], G, -1)
        w = torch.softmax(torch.einsum("hgd,hld->hgl", qi, k[:, rows]) * st["scale"], -1)
        out.append(torch.einsum("hgl,hld->hgd", w, v[:, rows]).reshape(c["H"], -1))
    return torch.stack(out)
