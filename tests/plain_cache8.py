"""A cache in 8 bits and attention over it in plain 64-bit PyTorch, sharing no code with the kernels.

Blocks of 16 tokens hold e4m3 numbers under one power of two for each kv head: 2^e with the smallest e in -100 .. 119 for which the block's largest
magnitude is at most 448 * 2^e."""

import math

import torch

E4M3, F64, U8 = torch.float8_e4m3fn, torch.float64, torch.uint8
HALF_STEP = 2.0**-4  # an e4m3 rounding is off by at most this part of the number
SMALLEST_HALF_STEP = 2.0**-10  # and, under the smallest normal number, by at most this much, times the scale


def scale_of(amax: float) -> float:
    e = -100
    while e < 119 and amax > 448 * 2.0**e:
        e += 1
    return 2.0**e


def empty(num_pages, KV, bs, D, device="cpu"):
    """(k_pages, v_pages, k_scales, v_scales), zeroed."""
    nb = bs // 16
    return (torch.zeros(num_pages, KV, bs, D, dtype=U8, device=device).view(E4M3),
            torch.zeros(num_pages, KV, nb, D, 16, dtype=U8, device=device).view(E4M3),
            torch.zeros(num_pages, KV, nb, device=device), torch.zeros(num_pages, KV, nb, device=device))  # fmt: skip


def keys_of(pages, scales):
    """The keys [num_pages, KV, bs, D] that pages stand for, in 64 bits."""
    return pages.to(F64) * scales.to(F64).repeat_interleave(16, dim=2)[..., None]


def values_of(pages, scales):
    """The values [num_pages, KV, bs, D]."""
    v = pages.to(F64) * scales.to(F64)[..., None, None]
    return v.transpose(-1, -2).reshape(v.shape[0], v.shape[1], 16 * v.shape[2], v.shape[3])


def fill(cache, k, v):
    """Numbers k, v [num_pages, KV, bs, D] into a whole cache, every block at once."""
    k_pages, v_pages, k_scales, v_scales = cache
    P, KV, bs, D = k.shape
    for x, scales, values in ((k, k_scales, False), (v, v_scales, True)):
        x = x.to(F64).view(P, KV, bs // 16, 16, D)
        amax = x.abs().amax((-1, -2))
        s = torch.tensor([scale_of(a) for a in amax.flatten().tolist()], dtype=F64, device=x.device).view(amax.shape)
        scales.copy_(s)
        stored = (x / s[..., None, None]).float().to(E4M3).view(U8)
        if values:
            v_pages.view(U8).copy_(stored.transpose(-1, -2))
        else:
            k_pages.view(U8).copy_(stored.reshape(P, KV, bs, D))


def seen(position, length, window=0, keep=0, chunk=0):
    """Which of `length` keys a query sees."""
    key = torch.arange(length)
    ok = key <= position
    if chunk:
        ok &= key >= position // chunk * chunk
    if window:
        ok &= (key > position - window) | (key < keep)
    return ok


def attend(q, k, v, position, scale, window=0, keep=0, chunk=0, cap=0.0, sink=None):
    """One token: q [H, D], keys and values [KV, L, D] of its request.  Returns (out [H, D], bound [H, D]): `bound` is what the
    kernel's roundings may make of it."""
    H, D = q.shape
    KV, L, _ = k.shape
    q, k, v = q.to(F64), k.repeat_interleave(H // KV, 0).to(F64), v.repeat_interleave(H // KV, 0).to(F64)
    ok = seen(position, L, window, keep, chunk).to(q.device) if L else torch.zeros(0, dtype=torch.bool, device=q.device)
    if not bool(ok.any()):
        return torch.zeros(H, D, dtype=F64, device=q.device), torch.zeros(H, D, dtype=F64, device=q.device)
    k, v = k[:, ok], v[:, ok]
    s = (k @ q[..., None])[..., 0] * scale
    # A query's second part is off by 2^-10 of a scale of at most max / 224; sums of up to 512 products in 32 bits by 2^-24 a product, 2^-20 at most in all
    off = scale * ((q.abs().amax(-1, keepdim=True) * 2.0**-10 / 224) * k.abs().sum(-1) + 2.0**-20 * (k.abs() @ q.abs()[..., None])[..., 0])
    off = off.amax(-1, keepdim=True) + 2.0**-20 * s.abs().amax(-1, keepdim=True)
    if cap:
        s = cap * torch.tanh(s / cap)
        off = off + cap * 2.0**-21  # the hardware's exponential and reciprocal in tanh
    top = s.amax(-1, keepdim=True)
    if sink is not None:
        top = torch.maximum(top, sink.to(F64)[:, None])
    w = torch.exp(s - top)
    total = w.sum(-1, keepdim=True) + (torch.exp(sink.to(F64)[:, None] - top) if sink is not None else 0.0)
    out = (w[:, None] @ v)[:, 0] / total
    size = (w[:, None] @ v.abs())[:, 0] / total
    # Weights rounded to bfloat16, w (1 + e) with |e| <= 2^-8: with the sum of those that are not rounded as the denominator the result is off by
    # |sum w e v| / sum w <= 2^-8 size; with the sum of the rounded ones by |sum w e (v - out)| / sum w (1 + e), which is at most
    # 2^-8 (size + |out|) (1 + 2^-7).  The result is rounded once more, 2^-8 |out|.  Scores' errors count in numerator and denominator, sums are 32-bit.
    return out, 2.0**-8 * (1 + 2.0**-7) * (size + 2 * out.abs()) + (2 * off + 2.0**-16) * size + 1e-30


def gathered(cache, table, length):
    """Keys and values [KV, length, D] of one request; table: its page ids."""
    k_pages, v_pages, k_scales, v_scales = cache
    bs = k_pages.shape[2]
    pages = torch.as_tensor(table, device=k_pages.device).long()[: -(-length // bs)]
    k = keys_of(k_pages.view(U8)[pages].view(E4M3), k_scales[pages])
    v = values_of(v_pages.view(U8)[pages].view(E4M3), v_scales[pages])
    join = lambda x: x.transpose(0, 1).reshape(x.shape[1], x.shape[0] * x.shape[2], x.shape[3])[:, :length]  # noqa: E731
    return join(k), join(v)


def positions_angles(positions, rotary, theta=10000.0):
    inv = theta ** (-torch.arange(0, rotary, 2, dtype=F64) / rotary)
    a = torch.as_tensor(positions, dtype=F64)[:, None] * inv
    return torch.stack([a.cos(), a.sin()], -1).float()


def default_scale(D):
    return 1.0 / math.sqrt(D)
