"""4-bit key / value cache (omnicoder.ops.kv4): the format and its refusals on the CPU, the kernels
against the plain forms in 64 bits on the GPU, and the cache inside the model.

Tolerances.  Codes and parameters are whole numbers and stored bf16 values: equal.  Read-back: n * s
is exact in fp32, so the kernel's fused form and the plain one round the same number: equal.
Attention: with w the softmax weights, an output element is off by
    its own rounding                              eps / 2 * |o|
    the rounding of each weight times its scale   2^-11 * w * s * n in fp16, 2^-8 * w * s * |n - 8| in
                                                  bf16: both at most 2^-8 * w * 8 s
    the error ds of the scores, which changes each weight by a factor within 1 +- 2 ds:
        2 ds * sum w |v|,  ds = (W + 16) * 2^-23 * scale * max_t sum_d |q_d| (15 s + |m|)
        (fp32 sums of W products, none larger than that sum)
and, the roundings being independent of one another, its mean square by the sum of their squares.
"""
import math

import pytest
import torch

from omnicoder.ops import kv4
from omnicoder.ops.decode import decode_attention
from omnicoder.ops.kv4 import (decode_attention_kv4_torch, dequantize_kv4, kv4_alloc, kv4_group, kv4_read,
                               kv4_row_bytes, kv4_write, quantize_kv4)

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _rows(shape, seed, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * torch.exp(0.7 * torch.randn(shape[-1], generator=g))
    return x.to(dtype)


# ----------------------------------------------------------------------------------------------
# format
# ----------------------------------------------------------------------------------------------
def test_group_and_sizes():
    assert kv4_group(128) == 64 and kv4_group(576, 512) == 64 and kv4_group(192, 160) == 32
    assert kv4_group(176, 128) == 16 and kv4_group(32) == 32
    assert kv4_row_bytes(128) == 64 + 8 and kv4_row_bytes(576, 512) == 288 + 36
    for bad in (0, 24, 100):
        with pytest.raises(ValueError, match="multiple of 16"):
            kv4_group(bad)
    with pytest.raises(ValueError, match="value dims"):
        kv4_group(64, 40)
    c, p = kv4_alloc(2, 3, 33, 128)
    assert c.shape == (2, 3, 64, 64) and p.shape == (2, 3, 64, 2, 2)


def test_quantise_by_hand():
    """s = (15 - 0) / 15 = 1, ties to even, the group's ends exact, low nibble first."""
    x = torch.zeros(1, 16)
    x[0, :8] = torch.tensor([0.0, 15.0, 0.5, 1.5, 2.5, 7.49, 7.51, 14.5])
    codes, params = quantize_kv4(x, 16)
    assert params[0, 0].tolist() == [1.0, 0.0]
    n = torch.stack([codes & 15, codes >> 4], -1).reshape(-1)
    assert n[:8].tolist() == [0, 15, 0, 2, 2, 7, 8, 14] and n[8:].sum() == 0
    assert dequantize_kv4(codes, params).tolist()[0][:8] == [0, 15, 0, 2, 2, 7, 8, 14]


def _hard_rows(dtype):
    """[1, T, 1, 64] rows where a quantiser goes wrong."""
    inf, nan, tiny = float("inf"), float("nan"), 2.0 ** -130
    rows = [torch.zeros(64), torch.full((64,), -3.25), torch.linspace(-1, 1, 64)]
    r = torch.zeros(64)
    r[:5] = torch.tensor([-15.0, 15.0, 1e-9, -1e-9, 0.0])       # next to the border 7.5, from both sides and on it
    rows.append(r)
    r = torch.arange(64, dtype=torch.float32) / 2 - 16           # every border and every code
    rows.append(r)
    for bad in (inf, -inf, nan):
        r = torch.linspace(-1, 1, 64)
        r[17] = bad
        rows.append(r)
    rows.append(torch.arange(64) * tiny)                         # scale below 2^-120
    rows.append(torch.arange(64) * 2.0 ** -114)
    big = 60000.0 if dtype == torch.float16 else 3e38
    r = torch.zeros(64)
    r[0], r[1] = -big, big                                       # the range of fp32, or beyond it
    rows.append(r)
    return torch.stack(rows).to(dtype)[None, :, None, :].contiguous()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_hard_rows(device, dtype):
    x = _hard_rows(dtype)
    T = x.shape[1]
    codes, params = kv4_alloc(1, 1, T, 64, device=device)
    pos = torch.arange(T, device=device)[None]
    kv4_write(pos, x.to(device), codes, params)
    want_c, want_p = quantize_kv4(x, 64)
    assert torch.equal(codes.cpu()[0, 0, :T], want_c[0, :, 0])
    assert torch.equal(torch.nan_to_num(params.cpu()[0, 0, :T], nan=7.0), torch.nan_to_num(want_p[0, :, 0], nan=7.0))
    back = kv4_read(pos, codes, params, dtype=torch.float32).cpu()[0, :, 0]
    assert torch.equal(back[0], torch.zeros(64)) and torch.equal(back[1], torch.full((64,), -3.25))
    assert torch.isnan(back[5:8]).all() and torch.isfinite(back[:5]).all()
    # half a step, and what rounding m and s to bf16 moves (x itself is off the grid of m by 2^-8 |m|)
    xf, s, m = x[0, :5, 0].float(), want_p[0, :5, 0, 0, 0].float()[:, None], want_p[0, :5, 0, 0, 1].float()[:, None]
    assert ((back[:5] - xf).abs() <= 0.5 * s + 2 ** -8 * (m.abs() + 16 * s)).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_values_far_below_a_border(device, dtype):
    """x - m is half a step away from a code but for an x that no 64-bit difference keeps: rounded as
    the exact quotient, taken in fractions.  Borders k + 1/2 with k even and odd, s = 2^p."""
    from fractions import Fraction
    top = 12 if dtype == torch.float16 else 100
    rows = []
    for p in (0, -3, top):                             # m = -(k + 1/2) s, max = m + 15 s, both exact in bf16
        for k in range(0, 15):
            s = 2.0 ** p
            r = torch.zeros(64, dtype=torch.float64)
            r[0], r[1] = -(k + 0.5) * s, (14.5 - k) * s
            small = [2.0 ** -24] if dtype == torch.float16 else [2.0 ** e for e in (-20, -52, -60, -100, -126)]
            for i, t in enumerate(small):
                r[2 + 2 * i], r[3 + 2 * i] = t, -t
            rows.append(r)
    x = torch.stack(rows).to(dtype)[None, :, None, :].contiguous()
    T = x.shape[1]
    codes, params = kv4_alloc(1, 1, T, 64, device=device)
    pos = torch.arange(T, device=device)[None]
    kv4_write(pos, x.to(device), codes, params)
    n = torch.stack([codes & 15, codes >> 4], -1).reshape(-1, 64)[:T].cpu()
    for t in range(T):
        s, m = (Fraction(float(params[0, 0, t, 0, i])) for i in range(2))
        want = [min(15, max(0, round((Fraction(float(v)) - m) / s))) for v in x[0, t, 0]]      # ties to even
        assert n[t].tolist() == want, t


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_scale_is_the_product_with_a_fifteenth(device, dtype):
    """Ranges of 15 times an odd 9-bit number: the quotient by 15 lies halfway between two bf16 scales, the
    product with fp32(1 / 15) beside it.  The format takes the product."""
    q = torch.arange(257, 512, 2)
    R = 15 * q                                          # <= 7665: hi = its upper bits, lo = -(the rest)
    hi = R // 32 * 32
    x = torch.zeros(1, len(q), 1, 64)
    x[0, :, 0, 0], x[0, :, 0, 1] = hi.float(), (hi - R).float()
    codes, params = kv4_alloc(1, 1, len(q), 64, device=device)
    kv4_write(torch.arange(len(q), device=device)[None], x.to(dtype).to(device), codes, params)
    fifteenth = torch.tensor(1.0 / 15.0).double()       # fp32(1 / 15); the product of 13 and 24 bits is exact in 64
    want = (R.double() * fifteenth).float().to(torch.bfloat16)
    even = torch.where(q % 4 == 1, q - 1, q + 1).to(torch.bfloat16)
    assert torch.equal(params[0, 0, :len(q), 0, 0].cpu(), want)
    assert (want != even).sum() > 40                    # the quotient would round these to the other side


def _border_rows(n, dtype, seed):
    """[1, n, 1, 64] groups whose values lie on borders between codes or a few units of the last place
    beside them, next to the sizes at which the kernel decides in another way: minima of every size
    from 2^-20 of the range to 2^6 times it, values around 2^-16 of the range, scales down to 2^-100."""
    g = torch.Generator().manual_seed(seed)
    lo_e = (-3, 3) if dtype == torch.float16 else (-100, 100)
    size = 2.0 ** torch.randint(lo_e[0], lo_e[1] + 1, (n, 1), generator=g).double()
    R = (1 + torch.rand(n, 1, generator=g).double()) * size
    least = R * torch.randn(n, 1, generator=g).double().sign() * 2.0 ** torch.randint(-20, 7, (n, 1), generator=g).double()
    least = torch.where(torch.rand(n, 1, generator=g) < 0.5, -R * torch.rand(n, 1, generator=g).double(), least)
    least = torch.where(torch.rand(n, 1, generator=g) < 0.1, torch.zeros_like(least), least)
    x = torch.zeros(n, 64, dtype=torch.float64)
    x[:, 0], x[:, 1] = least[:, 0], least[:, 0] + R[:, 0]
    x = x.to(dtype)
    lo = x[:, :2].amin(-1).float()
    m = lo.to(torch.bfloat16).double()[:, None]
    s = ((x[:, :2].amax(-1).float() - m[:, 0].float()) * (1.0 / 15.0)).to(torch.bfloat16).double()[:, None]
    k = torch.randint(0, 15, (n, 62), generator=g).double()
    at = (m + (k + 0.5) * s).to(dtype)
    word = torch.int32 if dtype == torch.float32 else torch.int16
    near = (at.view(word) + torch.randint(-3, 4, (n, 62), generator=g).to(word)).view(dtype)
    tiny = (R * 2.0 ** -torch.randint(14, 40, (n, 62), generator=g).double() *
            torch.randn(n, 62, generator=g).double().sign()).to(dtype)
    pick = torch.where(torch.rand(n, 62, generator=g) < 0.15, tiny, near)
    hi = x[:, :2].amax(-1, keepdim=True)
    ok = torch.isfinite(pick) & (pick >= lo[:, None].to(dtype)) & (pick <= hi)       # the range stays
    x[:, 2:] = torch.where(ok, pick, x[:, :1].expand(-1, 62))
    return x[None, :, None, :].contiguous()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_plain_codes_next_to_borders(dtype):
    """The plain form against fractions."""
    from fractions import Fraction
    x = _border_rows(150, dtype, 80)
    codes, params = quantize_kv4(x, 64)
    n = torch.stack([codes & 15, codes >> 4], -1).reshape(-1, 64)
    for t in range(x.shape[1]):
        s, m = (Fraction(float(params[0, t, 0, 0, i])) for i in range(2))
        want = [min(15, max(0, round((Fraction(float(v)) - m) / s))) for v in x[0, t, 0]]
        assert n[t].tolist() == want, t


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("seed", [81, 82, 83])
def test_codes_next_to_borders(dtype, seed):
    """The kernel against the plain form: a million values, most of them within three units of the last
    place of a border."""
    x = _border_rows(1 << 14, dtype, seed)
    T = x.shape[1]
    codes, params = kv4_alloc(1, 1, T, 64, device="cuda")
    kv4_write(torch.arange(T, device="cuda")[None], x.cuda(), codes, params)
    want_c, want_p = quantize_kv4(x, 64)
    assert torch.equal(params[0, 0].cpu(), want_p[0, :, 0])
    assert torch.equal(codes[0, 0].cpu(), want_c[0, :, 0])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,T,Hk,W,latent", [(3, 5, 4, 128, 0), (2, 1, 1, 576, 512), (1, 33, 2, 64, 0), (2, 7, 1, 176, 128),
                                             (2, 3, 3, 32, 0), (1, 2, 1, 192, 160)])
def test_write_and_read(device, dtype, B, T, Hk, W, latent):
    """Keys and values in one launch, at scattered rows; rows that are not written stay as they were."""
    off, L = 4, 70
    k, v = _rows((B, T, Hk, W), 1, dtype), _rows((B, T, Hk, W), 2, dtype)
    g = torch.Generator().manual_seed(3)
    pos = torch.stack([torch.randperm(60, generator=g)[:T] for _ in range(B)])
    caches = [kv4_alloc(B, Hk, L, W, latent, device) for _ in range(2)]
    for c, p in caches:
        c.fill_(0xA5)
        p.fill_(0.5)
    (kc, kp), (vc, vp) = caches
    kv4_write(pos.to(device), k.to(device), kc, kp, v.to(device), vc, vp, row_offset=off)
    got = kv4_read(pos.to(device), kc, kp, vc, vp, row_offset=off, dtype=torch.float32)
    for x, (c, p), back in ((k, caches[0], got[0]), (v, caches[1], got[1])):
        want_c, want_p = quantize_kv4(x, kv4_group(W, latent))
        full_c, full_p = torch.full_like(c.cpu(), 0xA5), torch.full_like(p.cpu(), 0.5)
        for b in range(B):
            full_c[b, :, pos[b] + off] = want_c[b].transpose(0, 1)
            full_p[b, :, pos[b] + off] = want_p[b].transpose(0, 1)
        assert torch.equal(c.cpu(), full_c) and torch.equal(p.cpu(), full_p)
        assert torch.equal(back.cpu(), dequantize_kv4(want_c, want_p))
    one = kv4_read(pos.to(device).int(), kc, kp, row_offset=off, dtype=dtype)
    assert one.dtype == dtype and torch.equal(one.cpu(), got[0].cpu().to(dtype))


@pytest.mark.parametrize("device", DEVICES)
def test_rows_outside_the_cache(device):
    """Writes behind or before the cache are dropped, reads there are zeros; T = 0 does nothing."""
    x = _rows((1, 4, 2, 64), 4)
    c, p = kv4_alloc(1, 2, 32, 64, device=device)
    pos = torch.tensor([[-1, 0, 31, 32]], device=device)
    kv4_write(pos, x.to(device), c, p)
    back = kv4_read(pos, c, p).cpu()
    assert (back[0, 0] == 0).all() and (back[0, 3] == 0).all() and (back[0, 1] != 0).any() and (back[0, 2] != 0).any()
    assert (c[:, :, 1:31] == 0).all()
    kv4_write(pos[:, :0], x[:, :0].to(device), c, p)
    assert kv4_read(pos[:, :0], c, p).shape == (1, 0, 2, 64)


def test_refusals():
    c, p = kv4_alloc(2, 4, 32, 64)
    pos, x = torch.zeros(2, 1, dtype=torch.long), torch.zeros(2, 1, 4, 64)
    with pytest.raises(ValueError, match="does not fit"):
        kv4_write(pos, x[:, :, :3], c, p)
    with pytest.raises(ValueError, match="does not fit"):
        kv4_write(pos[:1], x, c, p)
    with pytest.raises(ValueError, match="codes must be"):
        kv4_write(pos, x, c.to(torch.int8), p)
    with pytest.raises(ValueError, match="params must be"):
        kv4_write(pos, x, c, p[:, :, :16])
    with pytest.raises(ValueError, match="params must be"):
        kv4_write(pos, x, c, None)
    with pytest.raises(ValueError, match="caches of their own"):
        kv4_write(pos, x, c, p, x, c, p)
    with pytest.raises(ValueError, match="groups of"):
        kv4_read(pos, *kv4_alloc(2, 4, 32, 128)[:1], torch.zeros(2, 4, 32, 1, 2, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="dtype"):
        kv4_read(pos, c, p, dtype=torch.int32)
    q, qp, n = torch.zeros(2, 1, 8, 64), torch.zeros(2, 1, dtype=torch.long), torch.ones(2, dtype=torch.int32)
    for args, kw, what in (
            ((q[:, :, :6], c, c, qp, n), {}, "against codes"),
            ((q, c, None, qp, n), {}, "v codes"),
            ((q, c, c, qp[:1], n), {}, "q_pos"),
            ((q, c, c, qp, n), {"sink_rows": 2, "n_sink": 3}, "n_sink"),
            ((q, c, c, qp, n), {"sink_rows": 64}, "n_sink"),
            ((q, c, c, qp, n), {"window": -1}, "window"),
            ((q, c, None, qp, n), {"latent_v_dim": 64}, "one head")):
        with pytest.raises(ValueError, match=what):
            decode_attention(*args, k_scale=p, v_scale=p, **kw)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("latent", [0, 64])
@pytest.mark.parametrize("B,rows,T", [(2, 0, 3), (0, 32, 3), (2, 32, 0), (0, 0, 0)])
def test_empty_calls(device, latent, B, rows, T):
    """A cache without rows reads as zeros and is attended as one that no query sees; no sequences, no
    tokens: nothing."""
    W, Hk = (128, 1) if latent else (64, 2)
    (kc, kp), (vc, vp) = (kv4_alloc(B, Hk, rows, W, latent, device) for _ in range(2))
    pos = torch.zeros(B, T, dtype=torch.long, device=device) + torch.arange(T, device=device)
    x = torch.ones(B, T, Hk, W, device=device)
    kv = (None, None, None) if latent else (x, vc, vp)
    kv4_write(pos, x, kc, kp, *kv)
    got = kv4_read(pos, kc, kp, *kv[1:])
    for y in (got if isinstance(got, tuple) else (got,)):
        assert y.shape == (B, T, Hk, W) and (y == (1 if rows else 0)).all()
    q = torch.ones(B, T, 4, W, dtype=torch.bfloat16, device=device)
    n = torch.full((B,), T, dtype=torch.int32, device=device)
    o = decode_attention(q, kc, kv[1], pos, n, k_scale=kp, v_scale=kv[2], latent_v_dim=latent)
    assert o.shape == (B, T, 4, latent or W) and (o == (1 if rows else 0)).all()


@pytest.mark.parametrize("device", DEVICES)
def test_one_tensor_for_keys_and_values_is_refused(device):
    """Codes or parameters that k and v would both write; heads of one allocation are fine."""
    (kc, kp), (vc, vp) = (kv4_alloc(1, 2, 32, 64, device=device) for _ in range(2))
    pos, x = torch.zeros(1, 1, dtype=torch.long, device=device), torch.ones(1, 1, 2, 64, device=device)
    for pair in ((kc, vp), (vc, kp), (kc, kp)):
        with pytest.raises((ValueError, RuntimeError), match="caches of their own"):
            kv4_write(pos, x, kc, kp, x, *pair)
    assert (kc == 0).all() and (kp == 0).all()
    c, p = kv4_alloc(1, 4, 32, 64, device=device)
    kv4_write(pos, x, c[:, :2], p[:, :2], 2 * x, c[:, 2:], p[:, 2:])
    assert p[0, :, 0, 0, 1].tolist() == [1, 1, 2, 2]


# ----------------------------------------------------------------------------------------------
# attention
# ----------------------------------------------------------------------------------------------
def _cache(B, Hk, L, W, latent, seed, device):
    c, p = kv4_alloc(B, Hk, L, W, latent, device)
    kv4_write(torch.arange(c.shape[2], device=device).expand(B, -1), _rows((B, c.shape[2], Hk, W), seed).to(device), c, p)
    return c, p


def _bound(q, kc, kp, vc, vp, q_pos, kv_len, latent, out, kw):
    """(worst, mean square) of the error that the docstring of this file derives."""
    args = dict(kw, k_params=kp, v_params=vp, latent_v_dim=latent)
    qd = q.double()
    want = decode_attention_kv4_torch(qd, kc, vc, q_pos, kv_len, **args)
    sc, sp = (kc, kp) if latent else (vc, vp)
    g = 2 * sc.shape[-1] // sp.shape[3]
    V = latent or 2 * sc.shape[-1]

    def weigh(value, power=1):
        """sum_t w^power * value over the rows that a query sees."""
        Hk = kc.shape[1]
        vals = value.double().repeat_interleave(g, -1)[..., :V] if value.shape[-1] != V else value.double()
        B, Tn, H, W = q.shape
        kf = dequantize_kv4(kc, kp, torch.float64)
        qf = qd.reshape(B, Tn, Hk, H // Hk, W).permute(0, 2, 1, 3, 4).reshape(B, Hk, -1, W)
        s = torch.matmul(qf, kf.transpose(-1, -2)) * kw["scale"]
        rows = torch.arange(kc.shape[2], device=q.device)
        pp, t = rows - kw["sink_rows"], q_pos.long()[:, :, None]
        seen = (pp >= 0) & (pp < kv_len.long()[:, None, None]) & (pp <= t)
        if kw["window"]:
            seen &= pp > t - kw["window"]
        seen |= rows < kw["n_sink"]
        seen = seen[:, None, :, None].expand(B, Hk, Tn, H // Hk, -1).reshape(s.shape)
        w = torch.nan_to_num(torch.softmax(s.masked_fill(~seen, float("-inf")), -1)) ** power
        o = torch.matmul(w, vals)
        return o.reshape(B, Hk, Tn, H // Hk, -1).permute(0, 2, 1, 3, 4).reshape(B, Tn, H, -1)

    scales = sp[..., 0].double()
    vf = dequantize_kv4(sc, sp, torch.float64)[..., :V]
    kmag = (15 * kp[..., 0].double() + kp[..., 1].double().abs()).repeat_interleave(2 * kc.shape[-1] // kp.shape[3], -1)
    top = kmag.amax(2).repeat_interleave(q.shape[2] // kc.shape[1], 1)                     # [B, H, W]
    ds = (q.shape[3] + 16) * 2.0 ** -23 * abs(kw["scale"]) * (qd.abs() * top[:, None]).sum(-1, keepdim=True)
    half = torch.finfo(q.dtype).eps / 2
    worst = half * want.abs() + 2.0 ** -8 * weigh(8 * scales) + 2 * ds * weigh(vf.abs()) + 1e-30
    square = (half * want) ** 2 + 2.0 ** -16 * weigh((8 * scales) ** 2, 2)
    return want, worst, square


def _check_attention(q, kc, kp, vc, vp, q_pos, kv_len, latent=0, **kw):
    kw = {"window": 0, "sink_rows": 0, "n_sink": 0, "scale": 1 / math.sqrt(q.shape[-1]), **kw}
    out = decode_attention(q, kc, vc, q_pos, kv_len, k_scale=kp, v_scale=vp, latent_v_dim=latent, **kw)
    want, worst, square = _bound(q, kc, kp, vc, vp, q_pos, kv_len, latent, out, kw)
    assert out.shape == want.shape and out.dtype == q.dtype
    err = (out.double() - want).abs()
    assert (err <= worst).all(), float((err / worst).max())
    assert float((err ** 2).mean()) <= float(square.mean()) + 1e-30
    return out, want


def _attend_case(B, Tn, H, Hk, W, latent, ctx, seed, device="cuda", dtype=torch.bfloat16, sink=0, lens=None):
    L = sink + ctx
    kc, kp = _cache(B, Hk, L, W, latent, seed, device)
    vc, vp = (None, None) if latent else _cache(B, Hk, L, W, 0, seed + 1, device)
    q = _rows((B, Tn, H, W), seed + 2, dtype).to(device)
    g = torch.Generator().manual_seed(seed + 3)
    kv_len = (torch.randint(Tn, ctx + 1, (B,), generator=g) if lens is None else torch.tensor(lens)).int().to(device)
    q_pos = kv_len.long()[:, None] - Tn + torch.arange(Tn, device=device)[None]
    return q, kc, kp, vc, vp, q_pos, kv_len


HEADS = [(48, 8, 128, 0), (8, 8, 128, 0), (16, 2, 64, 0), (3, 1, 128, 0), (4, 4, 32, 0), (12, 2, 96, 0), (2, 1, 16, 0),
         (16, 1, 576, 512), (16, 1, 320, 256), (8, 1, 192, 160), (8, 1, 176, 128), (5, 1, 576, 512)]


@pytest.mark.gpu
@pytest.mark.parametrize("H,Hk,W,latent", HEADS)
@pytest.mark.parametrize("Tn", [1, 5])
@pytest.mark.parametrize("ctx", [5, 31, 129, 700])
def test_attention(H, Hk, W, latent, Tn, ctx):
    _check_attention(*_attend_case(3, Tn, H, Hk, W, latent, ctx, seed=ctx + Tn), latent=latent)


@pytest.mark.gpu
@pytest.mark.parametrize("H,Hk,W,latent", HEADS)
@pytest.mark.parametrize("window,sink,n_sink", [(1, 0, 0), (100, 0, 0), (0, 7, 7), (33, 40, 37), (300, 64, 0)])
def test_attention_window_and_memory(H, Hk, W, latent, window, sink, n_sink):
    case = _attend_case(4, 3, H, Hk, W, latent, 500, seed=7, sink=sink, lens=[3, 500, 64, 257])
    _check_attention(*case, latent=latent, window=window, sink_rows=sink, n_sink=n_sink)


@pytest.mark.gpu
@pytest.mark.parametrize("H,Hk,W,latent", [(48, 8, 128, 0), (16, 2, 64, 0), (4, 4, 32, 0), (16, 1, 576, 512), (16, 1, 320, 256)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_attention_long_and_many_rows(H, Hk, W, latent, dtype):
    """Splits of a long context, and more new tokens than one block of query rows."""
    _check_attention(*_attend_case(1, 1, H, Hk, W, latent, 6001, seed=11, dtype=dtype), latent=latent)
    _check_attention(*_attend_case(2, 19, H, Hk, W, latent, 300, seed=12, dtype=dtype), latent=latent)


@pytest.mark.gpu
@pytest.mark.parametrize("H,Hk,W,latent", HEADS)
def test_attention_rows_that_see_nothing(H, Hk, W, latent):
    """kv_len 0, positions before the cache, a window that has moved past the end: zeros, and the
    other queries of the call as usual."""
    q, kc, kp, vc, vp, q_pos, kv_len = _attend_case(4, 2, H, Hk, W, latent, 200, seed=13, lens=[0, 50, 100, 150])
    q_pos = torch.tensor([[0, 1], [-5, 49], [400, 99], [148, 149]], device="cuda")
    out, _ = _check_attention(q, kc, kp, vc, vp, q_pos, kv_len, latent=latent, window=120)
    assert (out[0] == 0).all() and (out[1, 0] == 0).all() and (out[2, 0] == 0).all()
    assert (out[1, 1] != 0).any() and (out[2, 1] != 0).any()


@pytest.mark.gpu
@pytest.mark.parametrize("H,Hk,W,latent", HEADS)
def test_attention_ignores_what_it_does_not_see(H, Hk, W, latent):
    """NaN and infinite parameters in rows behind the sequence, before the window, in unused memory
    rows and at positions that only a later query sees."""
    q, kc, kp, vc, vp, q_pos, kv_len = _attend_case(2, 3, H, Hk, W, latent, 400, seed=14, sink=16, lens=[301, 77])
    kw = dict(latent=latent, window=50, sink_rows=16, n_sink=5)
    clean, _ = _check_attention(q, kc, kp, vc, vp, q_pos, kv_len, **kw)
    for p in (kp, vp):
        if p is None:
            continue
        for b, n in enumerate([301, 77]):
            p[b, :, 16 + n:] = float("nan")
            p[b, :, 5:16] = float("inf")
            p[b, :, 16:16 + n - 3 - 50 + 1] = float("-inf")
            p[b, :, 16 + n - 1] = float("nan")             # the newest row: seen by the last query only
    out = decode_attention(q, kc, vc, q_pos, kv_len, k_scale=kp, v_scale=vp, latent_v_dim=latent, window=50,
                           sink_rows=16, n_sink=5)
    assert torch.equal(out[:, :2], clean[:, :2]) and torch.isnan(out[:, 2]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("H,Hk,W,latent", HEADS)
def test_attention_nan_of_one_group(H, Hk, W, latent):
    """A NaN among the values of one group of a row: the dims of that group, of the queries that see
    the row, and nothing else (latent rows are keys too: there the whole query)."""
    q, kc, kp, vc, vp, q_pos, kv_len = _attend_case(2, 3, H, Hk, W, latent, 200, seed=17, lens=[150, 60])
    kw = dict(scale=W ** -0.5, latent_v_dim=latent)
    clean = decode_attention(q, kc, vc, q_pos, kv_len, k_scale=kp, v_scale=vp, **kw)
    g = W // kp.shape[3]
    (kp if latent else vp)[0, :, 149, 0] = float("nan")        # seen by the last query of sequence 0
    out = decode_attention(q, kc, vc, q_pos, kv_len, k_scale=kp, v_scale=vp, **kw)
    bad = torch.zeros_like(out, dtype=torch.bool)
    bad[0, 2, :, :(out.shape[3] if latent else g)] = True
    assert torch.equal(torch.isnan(out), bad) and torch.equal(out[~bad], clean[~bad])


@pytest.mark.gpu
@pytest.mark.parametrize("H,Hk,W,latent", HEADS)
@pytest.mark.parametrize("window", [0, 40])
def test_attention_of_huge_queries(H, Hk, W, latent, window):
    """Queries of 2^122 against keys of 2^-118 beside queries of usual size and of zeros: the scores are
    of usual size, but no single fp32 factor takes a normalised query's product to them."""
    q, kc, kp, vc, vp, q_pos, kv_len = _attend_case(3, 2, H, Hk, W, latent, 400, seed=31, lens=[400, 1, 257])
    g = W // kp.shape[3]
    if latent:                               # small keys in the dims that are not the value
        q[..., :latent] = 0
        kp[:, :, :, latent // g:] *= 2.0 ** -118
    else:
        kp *= 2.0 ** -118
    q *= 2.0 ** 122
    q[1, 0] *= 2.0 ** -140
    q[2, 1, ::2] = 0
    out, _ = _check_attention(q, kc, kp, vc, vp, q_pos, kv_len, latent=latent, window=window, scale=W ** -0.5)
    assert torch.isfinite(out).all() and (out != 0).any()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("H,Hk,W", [(48, 8, 128), (8, 8, 128), (16, 2, 64), (4, 4, 32), (12, 2, 96)])
@pytest.mark.parametrize("row", [5, 70, 149])
def test_attention_nan_of_no_weight(device, H, Hk, W, row):
    """A NaN in a row that a query sees counts, however small the row's weight: in a tile that every
    query sees whole and in one that ends inside the sequence."""
    q, kc, kp, vc, vp, q_pos, kv_len = _attend_case(2, 2, H, Hk, W, 0, 200, seed=32, device=device, lens=[150, 60])
    kw = dict(scale=0.5, window=148)         # row 5 is seen by both queries of sequence 0
    q.zero_()
    q[..., 0] = 2.0
    kp[..., 0], kp[..., 1] = 0, 0            # scores 0, and -400 for the row
    kp[:, :, row, :, 1] = -400.0
    clean = decode_attention(q, kc, vc, q_pos, kv_len, k_scale=kp, v_scale=vp, **kw)
    assert torch.isfinite(clean).all()
    vp[0, :, row, 0] = float("nan")
    out = decode_attention(q, kc, vc, q_pos, kv_len, k_scale=kp, v_scale=vp, **kw)
    bad = torch.zeros_like(out, dtype=torch.bool)
    bad[0, (1 if row == 149 else 0):, :, :W // vp.shape[3]] = True
    assert torch.equal(torch.isnan(out), bad) and torch.equal(out[~bad], clean[~bad])


@pytest.mark.gpu
@pytest.mark.parametrize("H,Hk,W,latent", [(8, 8, 128, 0), (16, 1, 576, 512), (4, 4, 32, 0)])
def test_attention_extreme_values(H, Hk, W, latent):
    """Scores far apart, large and tiny queries, scales of very different size, one head of zeros."""
    q, kc, kp, vc, vp, q_pos, kv_len = _attend_case(2, 2, H, Hk, W, latent, 300, seed=15, lens=[300, 299])
    q[0] *= 2.0 ** 20
    q[1] *= 2.0 ** -60
    q[:, :, 0] = 0
    if vp is not None:
        vp[:, :, ::3] *= 2.0 ** 40
        vp[:, :, 1::3] *= 2.0 ** -40
    out = decode_attention(q, kc, vc, q_pos, kv_len, k_scale=kp, v_scale=vp, latent_v_dim=latent, scale=2.0 ** -18)
    want = decode_attention_kv4_torch(q.double(), kc, vc, q_pos, kv_len, k_params=kp, v_params=vp, latent_v_dim=latent,
                                      scale=2.0 ** -18)
    _check_attention(q, kc, kp, vc, vp, q_pos, kv_len, latent=latent, scale=2.0 ** -18)
    assert torch.isfinite(out).all() and torch.isfinite(want).all()


@pytest.mark.gpu
@pytest.mark.parametrize("H,Hk,W,latent", [(8, 8, 128, 0), (48, 8, 128, 0), (16, 2, 64, 0), (64, 4, 128, 0), (16, 1, 576, 512),
                                           (16, 1, 320, 256), (4, 4, 32, 0)])
@pytest.mark.parametrize("lens", [[130], [1], [40, 3, 0, 700, 128, 33, 1]])
@pytest.mark.parametrize("Tn", [1, 4])
def test_attention_in_a_cache_far_longer_than_the_text(H, Hk, W, latent, lens, Tn):
    """The host plans for the allocated rows, the device finds a few of them used."""
    case = _attend_case(len(lens), Tn, H, Hk, W, latent, 8192, seed=33, lens=lens)
    _check_attention(*case, latent=latent)


@pytest.mark.gpu
@pytest.mark.parametrize("H,Hk,W,latent", [(48, 8, 128, 0), (64, 4, 128, 0), (32, 8, 64, 0), (16, 1, 576, 512), (16, 1, 320, 256)])
def test_attention_rounds_weights_to_eleven_bits(H, Hk, W, latent):
    """Values of usual sizes meet weights p s in fp16.  A weight's rounding is off by at most 2^-11 w s n, and
    the roundings are independent: the mean square error is at most sum_t (2^-11 w s n)^2 and that of the
    output's own rounding, 2^-11 |o| in fp16.  The scores are single products here (2^-20 of a weight:
    a few fp32 roundings of scores up to 4 and the exponential's).  bf16 weights, 2^-8 w s |n - 8|, are
    worse than that; so the oracle with such weights has to be."""
    B, ctx = 64, 40
    lens = [2 + i % 39 for i in range(B)]
    q, kc, kp, vc, vp, q_pos, kv_len = _attend_case(B, 1, H, Hk, W, latent, ctx, seed=34, lens=lens, dtype=torch.float16)
    g, L = W // kp.shape[3], kc.shape[2]
    level = torch.randint(-128, 129, (L,), generator=torch.Generator().manual_seed(35)).cuda() / 32
    q.zero_()
    q[..., latent] = 2.0                                     # one dim against groups of one value: score = level
    kp[:, :, :, latent // g:, 0], kp[:, :, :, latent // g:, 1] = 0, level.to(torch.bfloat16)[None, None, :, None]
    out = decode_attention(q, kc, vc, q_pos, kv_len, k_scale=kp, v_scale=vp, latent_v_dim=latent, scale=0.5).double()
    sc, sp = (kc, kp) if latent else (vc, vp)
    V = latent or W
    w = torch.softmax(level.double() + torch.where(torch.arange(L, device="cuda") < kv_len[:, None], 0.0, -math.inf), -1)
    s = sp[..., 0].double().repeat_interleave(g, -1)[..., :V]
    n = torch.stack([sc & 15, sc >> 4], -1).reshape(*sc.shape[:3], -1)[..., :V].double()
    v = dequantize_kv4(sc, sp, torch.float64)[..., :V]
    at = lambda x: torch.einsum("bl,bhld->bhd", w, x).repeat_interleave(H // Hk, 1)[:, None]
    sq = lambda x: torch.einsum("bl,bhld->bhd", w ** 2, x ** 2).repeat_interleave(H // Hk, 1)[:, None]
    want = at(v)
    square = sq(2.0 ** -11 * s * n) + (2.0 ** -11 * want) ** 2 + (2.0 ** -19 * at(v.abs())) ** 2
    err = (out - want).abs()
    assert (err <= 2.0 ** -11 * (at(s * n) + want.abs()) * 1.001 + 2.0 ** -19 * at(v.abs())).all()
    assert float((err ** 2).mean()) <= float(square.mean())
    ws = w[:, None, :, None] * s
    coarse = ((ws.to(torch.bfloat16).double() - ws) * (n - 8)).sum(2)
    assert float((coarse ** 2).mean()) > 1.5 * float(square.mean())


@pytest.mark.gpu
@pytest.mark.parametrize("H,Hk,W,latent", [(8, 8, 128, 0), (48, 8, 128, 0), (4, 2, 64, 0), (16, 1, 576, 512), (16, 1, 320, 256)])
@pytest.mark.parametrize("far", [2.0 ** 9, 2.0 ** 40])
def test_attention_scales_far_apart(H, Hk, W, latent, far):
    """Neighbouring rows whose values differ by 2^9 (still one power of two for all) and 2^40 (not any
    more): the large ones carry weights of e^-120, the small ones the result; then the other way
    round, row after row and in long runs."""
    kw = dict(latent=latent, scale=0.5)
    for period, big_first in ((3, False), (3, True), (128, False), (128, True)):
        q, kc, kp, vc, vp, q_pos, kv_len = _attend_case(2, 2, H, Hk, W, latent, 700, seed=18, lens=[700, 333])
        big = (torch.arange(kc.shape[2], device="cuda") // max(1, period // 3)) % 3 == 0
        seen = ~big if not big_first else big
        level = torch.where(seen, 60.0, -60.0).to(torch.bfloat16)       # logits of the rows
        g = W // kp.shape[3]
        q.zero_()
        if latent:
            q[..., latent] = 2.0                                        # one rope dim against constant groups
            kp[:, :, :, latent // g:, 0], kp[:, :, :, latent // g:, 1] = 0, level[None, None, :, None]
            kp[:, :, big, :latent // g] *= far
        else:
            q[..., 0] = 2.0
            kp[..., 0], kp[..., 1] = 0, level[None, None, :, None]
            vp[:, :, big] *= far
        out, want = _check_attention(q, kc, kp, vc, vp, q_pos, kv_len, **kw)
        # weights of one size, at most 700: half a step of the output and 2^-8 of eight scales
        assert (out.double() - want).abs().max() <= 2.0 ** -7 * want.abs().max()


@pytest.mark.gpu
@pytest.mark.parametrize("H,Hk,W,latent", [(48, 8, 128, 0), (32, 8, 64, 0), (48, 4, 128, 0), (64, 4, 64, 0), (16, 1, 576, 512),
                                           (4, 1, 320, 256)])
@pytest.mark.parametrize("B,ctx,even,kw", [(61, 1100, False, {}), (64, 1100, True, {}), (260, 400, False, {}), (2, 3000, True, {}),
                                           (61, 3000, False, {}),
                                           (64, 1100, False, {"window": 700, "sink_rows": 40, "n_sink": 37})])
def test_attention_of_many_sequences(H, Hk, W, latent, B, ctx, even, kw):
    """Batches whose blocks walk several sequences, hold parts of one, or one each; then the same bits
    over NaN in every row that a sequence does not see."""
    g = torch.Generator().manual_seed(22)
    lens = [ctx] * B if even else [0, 1, ctx] + torch.randint(0, ctx + 1, (B - 3,), generator=g).tolist()
    sink = kw.get("sink_rows", 0)
    q, kc, kp, vc, vp, q_pos, kv_len = _attend_case(B, 1, H, Hk, W, latent, ctx, seed=23, lens=lens, sink=sink)
    want, _ = _check_attention(q, kc, kp, vc, vp, q_pos, kv_len, latent=latent, **kw)
    row = torch.arange(kc.shape[2], device="cuda")[None]
    unseen = (row >= kw.get("n_sink", 0)) & ((row < sink) | (row - sink >= kv_len[:, None]))
    for p in (kp, vp):
        if p is not None:
            p.masked_fill_(unseen[:, None, :, None, None], float("nan"))
    got = decode_attention(q, kc, vc, q_pos, kv_len, k_scale=kp, v_scale=vp, latent_v_dim=latent, **kw)
    assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("H,Hk,W,latent,B", [(48, 8, 128, 0, 12), (32, 8, 64, 0, 12), (16, 1, 576, 512, 100), (16, 1, 320, 256, 100)])
@pytest.mark.parametrize("long", [0, 5, -1])
def test_attention_of_one_long_sequence_among_short_ones(H, Hk, W, latent, B, long):
    """Fewer steps than blocks, most of them one sequence's."""
    lens = [1 + i % 3 for i in range(B)]
    lens[long] = 3900
    q, kc, kp, vc, vp, q_pos, kv_len = _attend_case(B, 1, H, Hk, W, latent, 4000, seed=26, lens=lens)
    _check_attention(q, kc, kp, vc, vp, q_pos, kv_len, latent=latent)


@pytest.mark.gpu
@pytest.mark.parametrize("H,W,latent", [(16, 320, 256), (16, 576, 512)])
@pytest.mark.parametrize("B,Tn", [(8, 4), (61, 1), (40, 6)])
def test_latent_blocks_that_walk_several_segments(H, W, latent, B, Tn):
    """Ragged drafted tokens: a block refills the stages in which its warps have just handed over their
    sums.  The same bits in every call, and no wait that ran out."""
    from omnicoder.ops import _ext
    g = torch.Generator().manual_seed(51)
    lens = torch.randint(Tn, 2100, (B,), generator=g).tolist()
    q, kc, kp, _, _, q_pos, kv_len = _attend_case(B, Tn, H, 1, W, latent, 2100, seed=52, lens=lens)
    first, _ = _check_attention(q, kc, kp, None, None, q_pos, kv_len, latent=latent)
    kw = dict(k_scale=kp, latent_v_dim=latent)
    outs = [decode_attention(q, kc, None, q_pos, kv_len, **kw) for _ in range(40)]
    assert all(torch.equal(o, first) for o in outs)
    _ext.check_status()


@pytest.mark.gpu
@pytest.mark.parametrize("H,Hk,W,latent", [(8, 1, 128, 0), (16, 1, 128, 0), (16, 1, 576, 512), (16, 1, 320, 256)])
@pytest.mark.parametrize("levels", [(40, -5, -50, -95), (-95, -50, -5, 40), (-60, 30, -60, 30), (40, -100, 40, -100),
                                    (-100, 40, -100, 40)])
def test_attention_scales_that_drop_and_rise(H, Hk, W, latent, levels):
    """Long runs of rows whose values are 2^level, all of one weight: the largest are the result.  260
    sequences, so that a block walks every run."""
    q, kc, kp, vc, vp, q_pos, kv_len = _attend_case(260, 1, H, Hk, W, latent, 1024, seed=24, lens=[1024] * 260)
    g, run = W // kp.shape[3], kc.shape[2] // len(levels)
    q.zero_()
    for n, e in enumerate(levels):
        (vp if vp is not None else kp[:, :, :, :latent // g])[:, :, n * run:(n + 1) * run] *= 2.0 ** e
    out, want = _check_attention(q, kc, kp, vc, vp, q_pos, kv_len, latent=latent)
    assert torch.isfinite(out).all()


@pytest.mark.gpu
@pytest.mark.parametrize("H,Hk,W,latent", [(8, 1, 128, 0), (16, 1, 576, 512), (16, 1, 320, 256)])
@pytest.mark.parametrize("s", [0.0, 2.0 ** -130])
def test_attention_of_constant_groups(H, Hk, W, latent, s):
    """Scales of zero, or below any that a quantised row has: the minima alone are the result."""
    q, kc, kp, vc, vp, q_pos, kv_len = _attend_case(2, 2, H, Hk, W, latent, 200, seed=25)
    kp[..., 0] = s
    if vp is not None:
        vp[..., 0] = s
    out, want = _check_attention(q, kc, kp, vc, vp, q_pos, kv_len, latent=latent)
    assert torch.isfinite(out).all()


@pytest.mark.gpu
@pytest.mark.parametrize("H,Hk,W,latent", [(8, 2, 128, 0), (16, 1, 576, 512), (4, 4, 32, 0)])
def test_attention_strides_streams_and_graphs(H, Hk, W, latent):
    """A slice of a larger batch with heads and sequences apart, int32 positions, a query that is a
    view, another stream, and a captured and replayed call: the same bits."""
    B, ctx = 3, 333
    q, kc, kp, vc, vp, q_pos, kv_len = _attend_case(B, 2, H, Hk, W, latent, ctx, seed=16)
    kw = dict(latent_v_dim=latent, window=200)
    want = decode_attention(q, kc, vc, q_pos, kv_len, k_scale=kp, v_scale=vp, **kw)

    def spread(t):
        if t is None:
            return None
        big = torch.full((2 * B, 2 * Hk) + tuple(t.shape[2:]), 3, dtype=t.dtype, device=t.device)
        big[1::2, ::2] = t
        return big[1::2, ::2]

    a = [spread(t) for t in (kc, vc, kp, vp)]
    wide = torch.randn(B, 2, H + 3, W, device="cuda").to(q.dtype)
    wide[:, :, :H] = q
    got = decode_attention(wide[:, :, :H], a[0], a[1], q_pos.int(), kv_len.long(), k_scale=a[2], v_scale=a[3], **kw)
    assert torch.equal(got, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = decode_attention(q, kc, vc, q_pos, kv_len, k_scale=kp, v_scale=vp, **kw)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graphs, outs = [], []
    for _ in range(2):                       # two graphs of one pool replayed in turn
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(decode_attention(q, kc, vc, q_pos, kv_len, k_scale=kp, v_scale=vp, **kw))
        graphs.append(g)
    for _ in range(2):
        for g, o in zip(graphs, outs):
            o.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(o, want)


_FIRST_CALL = """
import torch
from omnicoder.ops.decode import decode_attention
from omnicoder.ops.kv4 import kv4_alloc, kv4_write
H, Hk, W, latent = {shape}
caches = [kv4_alloc(2, Hk, 512, W, latent, "cuda") for _ in range(2)]
(kc, kp), (vc, vp) = caches if not latent else (caches[0], (None, None))
x = torch.randn(2, 512, Hk, W, device="cuda")
pos = torch.arange(512, device="cuda").expand(2, -1).contiguous()
q = torch.randn(2, 1, H, W, device="cuda").to(torch.bfloat16)
kv_len = torch.tensor([500, 20], dtype=torch.int32, device="cuda")
q_pos = kv_len.long()[:, None] - 1

def call():
    kv4_write(pos, x, kc, kp, None if latent else x, vc, vp)
    return decode_attention(q, kc, vc, q_pos, kv_len, k_scale=kp, v_scale=vp, latent_v_dim=latent)

g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    out = call()
g.replay()
torch.cuda.synchronize()
got = out.clone()
assert got.abs().max() > 0 and torch.equal(got, call())
print("captured first")
"""


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(8, 8, 128, 0), (16, 1, 576, 512), (4, 4, 32, 0)])
def test_the_first_call_of_a_process_is_captured(shape):
    import subprocess
    import sys
    from pathlib import Path
    r = subprocess.run([sys.executable, "-c", _FIRST_CALL.format(shape=shape)], cwd=Path(__file__).parents[1],
                       capture_output=True, text=True, timeout=240)
    assert r.returncode == 0 and "captured first" in r.stdout, r.stderr[-2000:]


@pytest.mark.gpu
@pytest.mark.parametrize("H,Hk,W,latent", HEADS)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_attention_of_one_bad_query(H, Hk, W, latent, bad):
    """A NaN or an infinity in one query row: that row is NaN, the others are as exact as ever.  (Not their
    bits: the running maximum of a block's rows moves when one row's has grown by 2^8, so a row that no
    longer calls for it changes where its neighbours' weights are rounded.)"""
    q, kc, kp, vc, vp, q_pos, kv_len = _attend_case(2, 2, H, Hk, W, latent, 300, seed=36)
    kw = dict(window=0, sink_rows=0, n_sink=0, scale=W ** -0.5)
    q_bad = q.clone()
    q_bad[1, 0, 0, 5] = bad
    out = decode_attention(q_bad, kc, vc, q_pos, kv_len, k_scale=kp, v_scale=vp, latent_v_dim=latent, **kw)
    assert torch.isnan(out[1, 0, 0]).all()
    want, worst, _ = _bound(q, kc, kp, vc, vp, q_pos, kv_len, latent, out, kw)
    out[1, 0, 0] = want[1, 0, 0].to(out.dtype)
    assert ((out.double() - want).abs() <= worst).all()


@pytest.mark.gpu
def test_calls_at_once():
    """Appends, read-backs and attention of two caches on two streams, interleaved without waiting: the
    bits of each alone."""
    def chain(c, out):
        q, kc, kp, vc, vp, q_pos, kv_len, latent, k, v = c
        for pos in range(3):
            at = kv_len.long()[:, None] - 1 - pos
            kv4_write(at, k, kc, kp, v, vc, vp)
            got = kv4_read(at, kc, kp, vc, vp)
            out += list(got) if isinstance(got, tuple) else [got]
            out.append(decode_attention(q, kc, vc, q_pos, kv_len, k_scale=kp, v_scale=vp, latent_v_dim=latent))

    cases = []
    for H, Hk, W, latent, seed in ((48, 8, 128, 0, 41), (16, 1, 576, 512, 42)):
        c = _attend_case(9, 1, H, Hk, W, latent, 1500, seed=seed)
        k = _rows((9, 1, Hk, W), seed + 5).cuda()
        cases.append((*c, latent, k, None if latent else k.flip(0).contiguous()))
    for c in cases:
        chain(c, [])                         # every row in place
    want = [[], []]
    for c, o in zip(cases, want):
        chain(c, o)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in cases], [[], []]
    for _ in range(8):
        for s, c, o in zip(streams, cases, got):
            with torch.cuda.stream(s):
                chain(c, o)
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert len(g) == 8 * len(w) and all(torch.equal(x, w[i % len(w)]) for i, x in enumerate(g))


@pytest.mark.gpu
@pytest.mark.parametrize("W,latent", [(128, 0), (320, 256)])
def test_offsets_beyond_32_bits(W, latent):
    """Codes of more than 2^31 bytes (and 2^32 for the wider row): the last rows are written, read and
    attended over."""
    rows = (1 << 25) + (1 << 24) if latent == 0 else 1 << 25
    kc = torch.zeros(1, 1, rows, W // 2, dtype=torch.uint8, device="cuda")
    kp = torch.zeros(1, 1, rows, W // 64, 2, dtype=torch.bfloat16, device="cuda")
    x = _rows((1, 64, 1, W), 21).cuda()
    pos = torch.arange(rows - 64, rows, device="cuda")[None]
    kv4_write(pos, x, kc, kp)
    codes, params = quantize_kv4(x.cpu(), 64)
    assert torch.equal(kc[0, 0, -64:].cpu(), codes[0, :, 0]) and torch.equal(kp[0, 0, -64:].cpu(), params[0, :, 0])
    assert torch.equal(kv4_read(pos, kc, kp, dtype=torch.float32).cpu(), dequantize_kv4(codes, params))
    q = _rows((1, 1, 4, W), 22).cuda()
    kw = dict(scale=W ** -0.5, window=40, latent_v_dim=latent)
    out = decode_attention(q, kc, None if latent else kc, torch.tensor([[rows - 1]], device="cuda"),
                           torch.tensor([rows], device="cuda"), k_scale=kp, v_scale=None if latent else kp, **kw)
    sc, sp = kc[:, :, -64:].contiguous(), kp[:, :, -64:].contiguous()
    small = decode_attention(q, sc, None if latent else sc, torch.tensor([[63]], device="cuda"),
                             torch.tensor([64], device="cuda"), k_scale=sp, v_scale=None if latent else sp, **kw)
    # the same rows lie at other places of their tiles: both within half an output step of 64 bits
    assert (out.float() - small.float()).abs().max() <= 2 ** -6 * small.float().abs().max()


@pytest.mark.gpu
def test_gpu_refusals():
    c, p = kv4_alloc(1, 2, 64, 64, device="cuda")
    q, qp, n = torch.zeros(1, 1, 2, 64, device="cuda"), torch.zeros(1, 1, dtype=torch.long, device="cuda"), \
        torch.ones(1, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="bf16 or fp16"):
        decode_attention(q, c, c, qp, n, k_scale=p, v_scale=p)
    q = q.to(torch.bfloat16)
    with pytest.raises(RuntimeError, match="multiple of 32"):
        decode_attention(q, c[:, :, :40].contiguous(), c[:, :, :40].contiguous(), qp, n, k_scale=p[:, :, :40].contiguous(),
                         v_scale=p[:, :, :40].contiguous())
    with pytest.raises(RuntimeError, match="contiguous"):
        decode_attention(q, c[:, :, ::2], c[:, :, ::2], qp, n, k_scale=p[:, :, ::2], v_scale=p[:, :, ::2])
    with pytest.raises(RuntimeError, match="device"):
        decode_attention(q, c, c, qp.cpu(), n, k_scale=p, v_scale=p)
    with pytest.raises(RuntimeError, match="positions"):
        kv4_write(qp.float(), torch.zeros(1, 1, 2, 64, device="cuda"), c, p)
    with pytest.raises(RuntimeError, match="share their rows"):
        kv4_write(qp.expand(2, 1), torch.zeros(2, 1, 2, 64, device="cuda"), c.expand(2, -1, -1, -1),
                  p.expand(2, -1, -1, -1, -1))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_writes_of_rows_that_were_just_made(dtype):
    """A write is set up while the kernel before it still makes its rows: read-backs of one cache into
    the next, and rows written over in place, without a pause."""
    src = [kv4_alloc(2, 2, 512, 64, device="cuda") for _ in range(4)]
    pos = torch.arange(512, device="cuda").expand(2, -1).contiguous()
    for i, (c, p) in enumerate(src):
        kv4_write(pos, _rows((2, 512, 2, 64), 60 + i).cuda(), c, p)
    want = [quantize_kv4(kv4_read(pos, c, p, dtype=dtype).cpu(), 64) for c, p in src]
    to = [kv4_alloc(2, 2, 512, 64, device="cuda") for _ in range(64)]
    for i, (c, p) in enumerate(to):
        kv4_write(pos, kv4_read(pos, *src[i % 4], dtype=dtype), c, p)
    for i, (c, p) in enumerate(to):
        assert torch.equal(c.cpu(), want[i % 4][0].transpose(1, 2)) and torch.equal(p.cpu(), want[i % 4][1].transpose(1, 2))
    x = torch.empty(2, 512, 2, 64, dtype=dtype, device="cuda")
    made = [_rows((2, 512, 2, 64), 70 + i, dtype).cuda() for i in range(4)]
    want = [quantize_kv4(m.cpu(), 64) for m in made]
    for i, (c, p) in enumerate(to):
        x.copy_(made[i % 4])
        kv4_write(pos, x, c, p)
    for i, (c, p) in enumerate(to):
        assert torch.equal(c.cpu(), want[i % 4][0].transpose(1, 2)) and torch.equal(p.cpu(), want[i % 4][1].transpose(1, 2))


@pytest.mark.gpu
def test_write_takes_views():
    """Keys and values as slices of a fused projection, without a copy or with one where they do not
    start on 16-byte boundaries."""
    fused = _rows((2, 3, 12, 64), 31).cuda()
    kc, kp = kv4_alloc(2, 4, 32, 64, device="cuda")
    vc, vp = kv4_alloc(2, 4, 32, 64, device="cuda")
    pos = torch.arange(3, device="cuda").expand(2, 3)
    kv4_write(pos, fused[:, :, 4:8], kc, kp, fused[:, :, 8:], vc, vp)
    for x, c, p in ((fused[:, :, 4:8], kc, kp), (fused[:, :, 8:], vc, vp)):
        codes, params = quantize_kv4(x.cpu(), 64)
        assert torch.equal(c[:, :, :3].cpu(), codes.transpose(1, 2)) and torch.equal(p[:, :, :3].cpu(), params.transpose(1, 2))
    odd = torch.zeros(2, 3, 4, 72, dtype=torch.bfloat16, device="cuda")[..., 1:65]
    odd.copy_(fused[:, :, :4])
    kv4_write(pos, odd, kc, kp)
    codes, params = quantize_kv4(fused[:, :, :4].cpu(), 64)
    assert torch.equal(kc[:, :, :3].cpu(), codes.transpose(1, 2)) and torch.equal(kp[:, :, :3].cpu(), params.transpose(1, 2))


# ----------------------------------------------------------------------------------------------
# the cache inside the model
# ----------------------------------------------------------------------------------------------
def _model(kind, device, dtype, window=0, mem=0, **attn):
    from omnicoder.config import AttentionConfig, ModelConfig, MoEConfig
    from omnicoder.models.lm import build_model
    a = AttentionConfig(kind=kind, window=window, mem_slots=mem, **attn)
    cfg = ModelConfig(name="kv4", vocab_size=512, d_model=256, n_layers=2, n_heads=4, ffn_dim=256, tie_embeddings=True,
                      max_seq_len=512, attn=a, moe=MoEConfig(n_experts=4, top_k=2, ffn_dim=128))
    return build_model(cfg, device=device, dtype=dtype, seed=0).eval()


KINDS = [("mha", {}), ("gqa", {"n_kv_heads": 2, "head_dim": 128}),
         ("mla", {"kv_lora_rank": 256, "qk_rope_dim": 64, "qk_nope_dim": 64, "v_head_dim": 64}),
         ("mla", {"kv_lora_rank": 128, "qk_rope_dim": 48, "qk_nope_dim": 48, "v_head_dim": 64})]


# the head sizes that the prompt's flash-attention kernel takes
GPU_KINDS = KINDS[:2] + [("mla", {"kv_lora_rank": r, "qk_rope_dim": 64, "qk_nope_dim": 64, "v_head_dim": 128})
                         for r in (256, 128)]


def _rounded_cache(cfg, B, rows, device):
    """A full-precision cache whose entries went through the 4-bit format."""
    from omnicoder.inference.kv_cache import KVCache

    class Rounded(KVCache):
        def write(self, layer, pos, k, v=None):
            g = kv4_group(self.k[0].shape[-1], self.cfg.attn.kv_lora_rank if self.mla else 0)
            super().write(layer, pos, *[None if x is None else dequantize_kv4(*quantize_kv4(x, g), dtype=x.dtype)
                                        for x in (k, v)])

        def view(self, b0, b1):
            v = super().view(b0, b1)
            v.__class__ = Rounded
            return v

    return Rounded(cfg, B, rows, device)


@pytest.mark.parametrize("kind,attn", KINDS)
def test_model_on_cpu(kind, attn):
    """Prompt, decode steps, a rolled-back token, memory rows: the logits of an int4 cache are those of
    an fp32 cache that holds the rounded entries (fp32 sums in another order: 1e-4 of the largest)."""
    from omnicoder.inference.kv_cache import KVCache
    m = _model(kind, "cpu", torch.float32, **attn)
    ids = torch.randint(0, 512, (3, 24), generator=torch.Generator().manual_seed(1))
    a, b = KVCache(m.cfg, 3, 40, "cpu", kv_dtype="int4"), _rounded_cache(m.cfg, 3, 40, "cpu")
    assert a.nbytes() <= 0.3 * b.nbytes()        # at most 6 of 32 bits (groups of 16), 64 rows for 40
    with torch.no_grad():
        for c in (a, b):
            c.out = [m.forward_cached(ids[:, :15], c, prefill=True)]
            c.out += [m.forward_cached(ids[:, i:i + 1], c) for i in range(15, 20)]
            c.rollback(c.lengths - torch.tensor([1, 0, 2]))
            c.out.append(m.forward_cached(ids[:, 20:23], c))
            c.reorder(torch.tensor([2, 0]))
            c.out.append(m.forward_cached(ids[:2, 23:], c))
            c.out.append(m.forward_cached(ids[:1, :1], c.view(1, 2)))
    for x, y in zip(a.out, b.out):
        assert (x - y).abs().max() <= 1e-4 * y.abs().max()
    k4, v4 = a.layer_kv(1)
    assert k4.shape[:2] == (2, 40) and (v4 is None) == a.mla
    assert torch.allclose(k4[:, :18], b.layer_kv(1)[0][:, :18], atol=1e-3)   # layer 1's inputs differ by fp32 sums


@pytest.mark.parametrize("kind,attn", KINDS)
def test_memory_rows_on_cpu(kind, attn):
    from omnicoder.inference.kv_cache import KVCache
    m = _model(kind, "cpu", torch.float32, window=8, mem=4, **attn)
    ids = torch.randint(0, 512, (2, 30), generator=torch.Generator().manual_seed(2))
    c = KVCache(m.cfg, 2, 40, "cpu", kv_dtype="int4")
    with torch.no_grad():
        m.forward_cached(ids[:, :29], c, prefill=True)
        before = c.layer_kv(0, torch.float32)
        assert c.compress_memory(8) == 4
        after = c.layer_kv(0, torch.float32)
        logits = m.forward_cached(ids[:, 29:], c)
    g = kv4_group(before[0].shape[-1], m.cfg.attn.kv_lora_rank if c.mla else 0)
    for x, y in zip(before, after):
        if x is None:
            continue
        bounds = [(i * 21) // 4 for i in range(5)]
        segs = torch.stack([x[:, 4 + s:4 + e].mean(1) for s, e in zip(bounds[:-1], bounds[1:])], 1)
        assert torch.equal(y[:, :4], dequantize_kv4(*quantize_kv4(segs, g)))
        assert torch.equal(y[:, 4:], x[:, 4:])
    assert torch.isfinite(logits).all()


def test_generate_and_budget_on_cpu():
    from omnicoder.config import get_preset
    from omnicoder.inference.generate import generate
    from omnicoder.inference.kv_cache import KVCache
    from omnicoder.inference.tools import estimate_memory
    from omnicoder.tools.utilities import kv_bytes_at
    m = _model("gqa", "cpu", torch.float32, n_kv_heads=2, head_dim=128)
    ids = torch.randint(0, 512, (2, 9), generator=torch.Generator().manual_seed(3))
    out = generate(m, ids, 6, temperature=0.0, kvq="int4")
    assert out.shape == (2, 15) and torch.equal(out[:, :9], ids)
    drafted = generate(m, ids, 6, temperature=0.0, kvq="int4", draft_model=_model("mha", "cpu", torch.float32),
                       speculative_draft_len=3)
    assert torch.equal(out, drafted)
    for name in ("dense_20b", "longctx_moe", "mobile_4gb"):
        cfg = get_preset(name)
        cfg.n_layers, cfg.attn.mem_slots = 2, 0
        c = KVCache(cfg, 3, 64, "cpu", kv_dtype="int4")
        assert c.nbytes() == kv_bytes_at(cfg, 64, "int4", batch=3) == estimate_memory(cfg, 3, 64, "int4")["kv_cache_bytes"]


@pytest.mark.gpu
@pytest.mark.parametrize("kind,attn", GPU_KINDS)
def test_model_on_gpu(kind, attn):
    """Prompt, eager steps, a captured and replayed step: write and attention together, against the
    bf16 cache that holds the rounded entries (both run bf16 layers: 2 % of the largest logit, the
    bound the bf16 cache itself is held to against the full forward pass is 5 %)."""
    from omnicoder.inference.graphs import GraphedStep
    from omnicoder.inference.kv_cache import KVCache
    m = _model(kind, "cuda", torch.bfloat16, **attn).prepare_inference()
    ids = torch.randint(0, 512, (3, 140), generator=torch.Generator().manual_seed(1)).cuda()
    a, b = KVCache(m.cfg, 3, 160, "cuda", kv_dtype="int4"), _rounded_cache(m.cfg, 3, 160, "cuda")
    a2 = KVCache(m.cfg, 3, 160, "cuda", kv_dtype="int4")
    with torch.no_grad():
        for c in (a, b, a2):
            c.out = [m.forward_cached(ids[:, :128], c, prefill=True, last_only=True)]
        step = GraphedStep(m, a2)
        for i in range(128, 134):
            for c in (a, b):
                c.out.append(m.forward_cached(ids[:, i:i + 1], c))
            a2.out.append(step(ids[:, i:i + 1]).clone())
        for c in (a, b, a2):
            c.out.append(m.forward_cached(ids[:, 134:139], c))
    for x, y, z in zip(a.out, b.out, a2.out):
        assert (x - y).abs().max() <= 2e-2 * y.abs().max()
        assert (z - x).abs().max() <= 2e-2 * x.abs().max()
    assert torch.equal(a.lengths, a2.lengths)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,attn", GPU_KINDS)
def test_generate_on_gpu(kind, attn):
    from omnicoder.inference.generate import generate
    m = _model(kind, "cuda", torch.bfloat16, window=96, mem=8, **attn)
    ids = torch.randint(0, 512, (2, 200), generator=torch.Generator().manual_seed(5)).cuda()
    out = generate(m, ids, 12, temperature=0.0, kvq="int4")
    assert out.shape == (2, 212) and torch.equal(out[:, :200], ids)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,attn", GPU_KINDS)
def test_speculative_decoding_on_gpu(kind, attn):
    """Several new tokens per step, and rejected ones that the next step writes over."""
    from omnicoder.inference.generate import generate
    m, draft = (_model(kind, "cuda", torch.bfloat16, **attn) for _ in range(2))
    ids = torch.randint(0, 512, (2, 100), generator=torch.Generator().manual_seed(6)).cuda()
    out, st = generate(m, ids, 10, temperature=0.0, kvq="int4", draft_model=draft, speculative_draft_len=3, return_stats=True)
    assert out.shape == (2, 110) and torch.equal(out[:, :100], ids)


def _one_layer(kind, seed=0, window=0, mem=0, **attn):
    """The entries of its cache depend on the embeddings alone, and its logits on the attention more than
    on anything else (another context changes them by as much as they are)."""
    from omnicoder.config import AttentionConfig, ModelConfig, MoEConfig
    from omnicoder.models.lm import build_model
    cfg = ModelConfig(name="kv4", vocab_size=512, d_model=256, n_layers=1, n_heads=4, ffn_dim=256, tie_embeddings=False,
                      max_seq_len=512, attn=AttentionConfig(kind=kind, window=window, mem_slots=mem, **attn),
                      moe=MoEConfig(n_experts=0))
    return build_model(cfg, device="cuda", dtype=torch.bfloat16, seed=seed).eval().prepare_inference()


def _check_tokens(m, out, S, first):
    """Every generated token is the largest logit, but for twice what the two caches' logits may differ by,
    of a cache that holds rounded entries and is given the same tokens: the entries in bf16, the
    attention's output, the projection, the layer's end and its norm, each off by 2^-8 at most, are 2 % of the
    largest logit.  first: prompt tokens of the first call."""
    import types

    from omnicoder.inference.kv_cache import KVCache
    B, T = out.shape
    c = _rounded_cache(m.cfg, B, T + 8, "cuda")
    g = kv4_group(c.k[0].shape[-1], m.cfg.attn.kv_lora_rank if c.mla else 0)

    def compress(self, window):
        n = KVCache.compress_memory(self, window)
        for t in [t for lst in (self.k, self.v) for t in lst if t is not None]:
            t[:, :self.sink] = dequantize_kv4(*quantize_kv4(t[:, :self.sink], g), dtype=t.dtype)
        return n

    c.compress_memory = types.MethodType(compress, c)
    with torch.no_grad():
        logits = [m.forward_cached(out[:, :first], c, prefill=True, last_only=True)]
        if m.cfg.attn.window and c.sink:
            assert c.compress_memory(m.cfg.attn.window) == c.sink
        logits += [m.forward_cached(out[:, i:i + 1], c) for i in range(first, T - 1)]
    y = torch.cat(logits, 1)[:, S - first:]                  # of the tokens out[:, S:]
    got = y.gather(-1, out[:, S:, None]).squeeze(-1)
    assert (got >= y.amax(-1) - 2 * 2e-2 * y.abs().amax()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind,attn", GPU_KINDS)
@pytest.mark.parametrize("window,mem", [(0, 0), (96, 8)])
def test_generated_tokens_on_gpu(kind, attn, window, mem):
    """Greedy tokens of an int4 cache, captured steps, with a window and memory rows."""
    from omnicoder.inference.generate import generate
    m = _one_layer(kind, window=window, mem=mem, **attn)
    ids = torch.randint(0, 512, (2, 200), generator=torch.Generator().manual_seed(7)).cuda()
    out = generate(m, ids, 12, temperature=0.0, kvq="int4")
    assert out.shape == (2, 212) and torch.equal(out[:, :200], ids)
    _check_tokens(m, out, 200, 200)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,attn", GPU_KINDS)
def test_rejected_drafts_on_gpu(kind, attn):
    """A draft model of other weights: most of its tokens are rejected, and the rows that they took in the
    cache are written over."""
    from omnicoder.inference.generate import generate
    m, draft = _one_layer(kind, **attn), _one_layer(kind, seed=1, **attn)
    ids = torch.randint(0, 512, (2, 100), generator=torch.Generator().manual_seed(8)).cuda()
    out, st = generate(m, ids, 12, temperature=0.0, kvq="int4", draft_model=draft, speculative_draft_len=3, return_stats=True)
    assert out.shape == (2, 112) and torch.equal(out[:, :100], ids)
    assert st.proposed_draft_tokens - st.accepted_draft_tokens >= 6
    _check_tokens(m, out, 100, 99)
