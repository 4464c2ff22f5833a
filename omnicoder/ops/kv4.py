"""4-bit key / value cache: append, read back and the attention that reads it.

A cache of one layer's keys (values have their own; an MLA latent is both):

    codes   uint8 [B, Hk, L, W / 2]      byte i of a row holds dim 2i (low nibble) and 2i + 1
    params  bf16  [B, Hk, L, W / g, 2]   (scale s, smallest value m) of each group of g dims

and stands for x = n * s + m, n = 0 .. 15.  A row of a head is contiguous, and so are the rows of a
head (head-major, unlike the bf16 / int8 cache): the attention kernels copy whole key tiles.  With
groups of 64 a value takes 4.5 bits (32: 5, 16: 6); an int8 cache of 128-wide heads takes 8.25.

Quantisation of a group: m = bf16(min x), s = bf16((max x - m) * (1 / 15)) with the product in fp32 (torch
on a GPU divides by 15 so, on a CPU it does not: quotients halfway between two bf16 numbers differ), and
n = clamp(round((x - m) / s), 0, 15), where the rounding (ties to even) is decided as if (x - m) / s
were exact.  s below 2^-120 is stored as 0 (then every n is 0 and the group reads back as m).  A group
that holds a NaN or an infinity, or whose range overflows fp32, reads back as NaN; other groups of
the row do not suffer.  The reference keeps 4-bit caches as nearest entries of a 16-value codebook
around mean and deviation (src/omnicoder/modeling/quant/kv_cache.py:108-257, omnicoder.quant.kv
here); equidistant codes turn a dot product with a group into one integer-valued dot product and two
multiplications, which is what a kernel needs that dequantises on its way to the tensor cores.

Position p of a sequence lives in row row_offset + p.  `kv4_write` skips positions whose row lies
outside the cache, `kv4_read` returns zeros for them.  The positions that one `kv4_write` call gives
for a sequence have to differ: two tokens written to one row at once leave a mixture.

CUDA: hand-written kernels (omnicoder/csrc/kv4*.cu; a call that does not fit raises RuntimeError; a
kernel whose copy never came gives NaN and omnicoder.ops._ext.check_status() raises);
CPU: the plain forms below (the oracle; ValueError).
"""
from __future__ import annotations

import math

import torch

from . import _ext

ROW_ALIGN = 32                       # rows of a cache: a multiple of the smallest key tile
_MIN_SCALE = 2.0 ** -120


def kv4_group(width: int, latent_v_dim: int = 0) -> int:
    """Dims per (scale, minimum) pair: the largest of 64, 32, 16 that divides the row width and, for
    a latent cache, the part of the row that is the value."""
    for g in (64, 32, 16):
        if width > 0 and width % g == 0 and latent_v_dim % g == 0:
            return g
    raise ValueError(f"a 4-bit cache needs rows of a multiple of 16 dims, got width {width}"
                     + (f" with {latent_v_dim} value dims" if latent_v_dim else ""))


def kv4_row_bytes(width: int, latent_v_dim: int = 0) -> int:
    """Bytes of one cached row (codes and parameters)."""
    return width // 2 + 4 * (width // kv4_group(width, latent_v_dim))


def kv4_alloc(batch: int, heads: int, rows: int, width: int, latent_v_dim: int = 0, device=None):
    """Zeroed (codes, params) for at least `rows` rows (rounded up to a multiple of 32)."""
    g = kv4_group(width, latent_v_dim)
    L = (rows + ROW_ALIGN - 1) // ROW_ALIGN * ROW_ALIGN
    return (torch.zeros(batch, heads, L, width // 2, dtype=torch.uint8, device=device),
            torch.zeros(batch, heads, L, width // g, 2, dtype=torch.bfloat16, device=device))


def _check_cache(codes, params, what: str):
    if codes.dtype != torch.uint8 or codes.dim() != 4:
        raise ValueError(f"{what}: codes must be uint8 [B, Hk, L, W / 2]")
    if params is None or params.dtype != torch.bfloat16 or params.dim() != 5 or params.shape[4] != 2 \
            or params.shape[:3] != codes.shape[:3]:
        raise ValueError(f"{what}: params must be bf16 [B, Hk, L, W / g, 2] beside codes {tuple(codes.shape)}")
    W, G = 2 * codes.shape[3], params.shape[3]
    if G == 0 or W % G or W // G not in (16, 32, 64):
        raise ValueError(f"{what}: groups of {W / max(G, 1):g} dims (16, 32 or 64)")
    if codes.device != params.device:
        raise ValueError(f"{what}: codes on {codes.device}, params on {params.device}")


# ----------------------------------------------------------------------------------------------
# plain forms
# ----------------------------------------------------------------------------------------------
def quantize_kv4(x: torch.Tensor, group: int):
    """x [..., W] -> (codes uint8 [..., W / 2], params bf16 [..., W / group, 2])."""
    g = x.double().reshape(*x.shape[:-1], x.shape[-1] // group, group)
    m = g.amin(-1).float().to(torch.bfloat16)
    s = ((g.amax(-1).float() - m.float()) * (1.0 / 15.0)).to(torch.bfloat16)
    bad = ~(torch.isfinite(g).all(-1) & torch.isfinite(m) & torch.isfinite(s))
    s = torch.where(s.float() < _MIN_SCALE, torch.zeros_like(s), s)
    md, sd = m.double()[..., None], s.double()[..., None]
    d = g - md                           # d + e = x - m exactly: an x far below m is not lost
    back = d - g
    e = (g - (d - back)) - (md + back)
    n = torch.round(d / sd)
    r, half, odd = d - n * sd, 0.5 * sd, n % 2 != 0
    n = n + ((r > half) | ((r == half) & ((e > 0) | ((e == 0) & odd)))).double()
    n = n - ((r < -half) | ((r == -half) & ((e < 0) | ((e == 0) & odd)))).double()
    n = n.clamp(0, 15)
    n = torch.where((bad | (s == 0))[..., None], torch.zeros_like(n), n).to(torch.uint8)
    n = n.reshape(*x.shape[:-1], x.shape[-1] // 2, 2)
    p = torch.stack([s, m], -1)
    p = torch.where(bad[..., None], torch.full_like(p, float("nan")), p)
    return n[..., 0] | (n[..., 1] << 4), p


def dequantize_kv4(codes: torch.Tensor, params: torch.Tensor, dtype=torch.float32) -> torch.Tensor:
    """codes [..., W / 2], params [..., W / g, 2] -> values [..., W]."""
    W = 2 * codes.shape[-1]
    n = torch.stack([codes & 15, codes >> 4], -1).reshape(*params.shape[:-1], W // params.shape[-2]).float()
    return (n * params[..., 0:1].float() + params[..., 1:2].float()).reshape(*codes.shape[:-1], W).to(dtype)


def decode_attention_kv4_torch(q, k, v, q_pos, kv_len, *, window=0, scale=None, k_params=None, v_params=None,
                               latent_v_dim=0, sink_rows=0, n_sink=0):
    """Dense masked softmax over the dequantised cache; rows that see nothing give zeros."""
    B, Tn, H, W = q.shape
    sc = scale if scale is not None else 1.0 / math.sqrt(W)
    Hk, L, G = k.shape[1], k.shape[2], H // k.shape[1]
    if L == 0 or q.numel() == 0:
        return q.new_zeros(B, Tn, H, latent_v_dim or W)
    ct = torch.float64 if q.dtype == torch.float64 else torch.float32
    kf = dequantize_kv4(k, k_params, ct)
    vf = kf[..., :latent_v_dim] if latent_v_dim else dequantize_kv4(v, v_params, ct)
    qf = q.to(ct).reshape(B, Tn, Hk, G, W).permute(0, 2, 1, 3, 4)                        # [B, Hk, Tn, G, W]
    s = torch.matmul(qf.reshape(B, Hk, -1, W), kf.transpose(-1, -2)) * sc               # [B, Hk, Tn * G, L]
    rows = torch.arange(L, device=q.device)
    p, t = rows - sink_rows, q_pos.long()[:, :, None]
    seen = (p >= 0) & (p < kv_len.long()[:, None, None]) & (p <= t)
    if window > 0:
        seen = seen & (p > t - window)
    seen = seen | (rows < n_sink)                                                        # [B, Tn, L]
    seen = seen[:, None, :, None].expand(B, Hk, Tn, G, L).reshape(s.shape)
    s = s.masked_fill(~seen, float("-inf"))
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(top == float("-inf"), torch.zeros_like(top), top))
    w = e / e.sum(-1, keepdim=True).masked_fill(~seen.any(-1, keepdim=True), 1.0)
    finite = torch.isfinite(vf)
    o = torch.matmul(w, torch.where(finite, vf, torch.zeros_like(vf)))
    if not bool(finite.all()):                     # a NaN counts for the queries that see its row
        o = o.masked_fill(torch.matmul(seen.to(ct), (~finite).to(ct)) > 0, float("nan"))
    return o.reshape(B, Hk, Tn, G, -1).permute(0, 2, 1, 3, 4).reshape(B, Tn, H, -1).to(q.dtype)


# ----------------------------------------------------------------------------------------------
# operators
# ----------------------------------------------------------------------------------------------
def kv4_write(pos, k, k_codes, k_params, v=None, v_codes=None, v_params=None, row_offset: int = 0) -> None:
    """Quantise new rows k (and v) [B, T, Hk, W] into the cache rows row_offset + pos[b, t], one launch
    for both.  pos int64 [B, T]; k and v fp32, fp16 or bf16."""
    if k.is_cuda:                        # checked by the bindings
        _ext.load().kv4_write(pos, k, k_codes, k_params, v, v_codes, v_params, row_offset)
        return
    if (v is None) != (v_codes is None):
        raise ValueError("kv4_write: v together with its cache")
    pairs = [(k, k_codes, k_params, "k")] + ([(v, v_codes, v_params, "v")] if v is not None else [])
    for x, c, p, what in pairs:
        _check_cache(c, p, f"kv4_write: {what}")
        if x.device != c.device:
            raise ValueError(f"kv4_write: {what} on {x.device}, its cache on {c.device}")
        if x.dim() != 4 or tuple(x.shape[:2]) != tuple(pos.shape) or x.shape[0] != c.shape[0] \
                or x.shape[2] != c.shape[1] or x.shape[3] != 2 * c.shape[3]:
            raise ValueError(f"kv4_write: {what} {tuple(x.shape)} does not fit positions {tuple(pos.shape)} and codes "
                             f"{tuple(c.shape)}")
    if v is not None and (v_codes.data_ptr() == k_codes.data_ptr() != 0 or v_params.data_ptr() == k_params.data_ptr() != 0):
        raise ValueError("kv4_write: k and v need caches of their own")
    rows = pos.long() + row_offset
    for x, c, p, _ in pairs:
        codes, params = quantize_kv4(x, x.shape[3] // p.shape[3])
        ok = (rows >= 0) & (rows < c.shape[2])
        b = torch.arange(rows.shape[0], device=rows.device)[:, None].expand_as(rows)[ok]
        c[b, :, rows[ok]] = codes[ok]
        p[b, :, rows[ok]] = params[ok]


def kv4_read(pos, k_codes, k_params, v_codes=None, v_params=None, row_offset: int = 0, dtype=torch.bfloat16):
    """Values [B, T, Hk, W] of the cache rows row_offset + pos[b, t]: k, or (k, v) when both are given.
    dtype: float32, float16 or bfloat16."""
    if dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise ValueError(f"kv4_read: dtype {dtype}")
    if k_codes.is_cuda:                  # checked by the bindings
        out = _ext.load().kv4_read(pos, k_codes, k_params, v_codes, v_params, row_offset, dtype)
        return tuple(out) if v_codes is not None else out[0]
    pairs = [(k_codes, k_params, "k")] + ([(v_codes, v_params, "v")] if v_codes is not None else [])
    for c, p, what in pairs:
        _check_cache(c, p, f"kv4_read: {what}")
        if pos.dim() != 2 or pos.shape[0] != c.shape[0]:
            raise ValueError(f"kv4_read: positions {tuple(pos.shape)} for codes {tuple(c.shape)}")
    rows = pos.long() + row_offset
    out = []
    for c, p, _ in pairs:
        ok = (rows >= 0) & (rows < c.shape[2])
        if c.shape[2] == 0:
            out.append(torch.zeros(*pos.shape, c.shape[1], 2 * c.shape[3], dtype=dtype, device=c.device))
            continue
        safe = torch.where(ok, rows, torch.zeros_like(rows))
        b = torch.arange(rows.shape[0], device=rows.device)[:, None].expand_as(rows)
        x = dequantize_kv4(c[b, :, safe], p[b, :, safe], dtype)
        out.append(torch.where(ok[:, :, None, None], x, torch.zeros_like(x)))
    return tuple(out) if v_codes is not None else out[0]


def decode_attention_kv4(q, k, v, q_pos, kv_len, *, window=0, scale=None, k_params=None, v_params=None,
                         latent_v_dim=0, sink_rows=0, n_sink=0):
    """Attention of new tokens q [B, Tn, H, W] against a 4-bit cache (k, v codes; v None with
    latent_v_dim = r for an MLA latent, whose value is the first r dims of a row).  Visibility as in
    omnicoder.ops.decode; a query that sees no row gets zeros.  |q| scale and scores up to 2^127.  Sums
    are fp32 in units of the largest scale of a head's rows: values up to 2^100, and of rows whose
    scales differ by more than 2^90 the smaller ones may be lost.  -> [B, Tn, H, W or r]."""
    sc = scale if scale is not None else 1.0 / math.sqrt(q.shape[3])
    if q.is_cuda:                        # checked by the bindings
        return _ext.load().kv4_attend(q, k, k_params, v, v_params, q_pos, kv_len, window, sc, latent_v_dim,
                                      sink_rows, n_sink)
    _check_cache(k, k_params, "decode_attention: k")
    if q.dim() != 4 or q.shape[0] != k.shape[0] or q.shape[3] != 2 * k.shape[3] or k.shape[1] == 0 \
            or q.shape[2] % k.shape[1]:
        raise ValueError(f"decode_attention: q {tuple(q.shape)} against codes {tuple(k.shape)}")
    if latent_v_dim:
        if v is not None or k.shape[1] != 1 or not 0 < latent_v_dim <= q.shape[3] \
                or latent_v_dim % (q.shape[3] // k_params.shape[3]):
            raise ValueError("decode_attention: a latent cache has one head, no v, and whole groups as its value")
    else:
        if v is None:
            raise ValueError("decode_attention: v codes, or latent_v_dim")
        _check_cache(v, v_params, "decode_attention: v")
        if v.shape != k.shape or v_params.shape != k_params.shape:
            raise ValueError("decode_attention: k and v caches of one shape")
    if tuple(q_pos.shape) != tuple(q.shape[:2]) or tuple(kv_len.shape) != (q.shape[0],):
        raise ValueError("decode_attention: q_pos [B, Tn], kv_len [B]")
    if not 0 <= n_sink <= sink_rows <= k.shape[2] or window < 0:
        raise ValueError("decode_attention: 0 <= n_sink <= sink_rows <= L, window >= 0")
    return decode_attention_kv4_torch(q, k, v, q_pos, kv_len, window=window, scale=sc, k_params=k_params,
                                      v_params=v_params, latent_v_dim=latent_v_dim, sink_rows=sink_rows,
                                      n_sink=n_sink)
