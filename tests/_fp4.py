"""The cache in 4 bits on the CPU: values to codes and back by their definition, in 64 bits."""
import torch

MAG = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
# every scale: the upper byte of an fp16
SCALES = (torch.arange(256) << 8).to(torch.int16).view(torch.float16).double()
USED = SCALES[:0x72]  # 0 .. 10240


def _nearest(x, table):
    """Index of the nearest entry of an ascending table, the even one in the middle."""
    i = torch.searchsorted(table, x.contiguous()).clamp(1, len(table) - 1)
    lo, hi = x - table[i - 1], table[i] - x
    return torch.where((hi < lo) | ((hi == lo) & (i % 2 == 0)), i, i - 1)


def encode(x):
    """Codes [..., D] and scale bytes [..., D / 32] of x, rounded to fp32 first."""
    g = x.float().double().unflatten(-1, (-1, 32))
    most = g.abs().amax(-1)
    fine = torch.isfinite(g).all(-1)
    s = _nearest((most.nan_to_num(0, posinf=0) / 6).clamp_max(10240), USED)
    f = USED[s].unsqueeze(-1)
    y = torch.where(f > 0, g.abs().nan_to_num(0, posinf=0) / f.clamp_min(1e-30), 0.0).clamp_max(6)
    c = _nearest(y, MAG) + 8 * torch.signbit(g).int()
    return c.flatten(-2).byte(), torch.where(fine, s, 0x7F).byte()


def decode(codes, scales):
    c = codes.int()
    v = MAG[c % 8] * torch.where(c >= 8, -1.0, 1.0)
    return (v.unflatten(-1, (-1, 32)) * SCALES[scales.int()].unsqueeze(-1)).flatten(-2)


def unpack(cache, is_v):
    """Codes [pages, heads, page, D] and scales [pages, heads, page, D / 32] of a cache."""
    P, H, page, row = cache.shape
    D = row // 17 * 32
    flat = cache.cpu().reshape(P, H, -1)
    c, s = flat[..., :page * D // 2], flat[..., page * D // 2:]
    c = torch.stack((c & 15, c >> 4), -1)
    if is_v:
        return (c.reshape(P, H, page // 8, D, 8).transpose(3, 4).reshape(P, H, page, D),
                s.reshape(P, H, page // 8, D // 32, 8).transpose(3, 4).reshape(P, H, page, D // 32))
    return c.reshape(P, H, page, D), s.reshape(P, H, page, D // 32)


def pack(codes, scales, is_v):
    """The cache [pages, heads, page, 17 D / 32] that holds these."""
    P, H, page, D = codes.shape
    if is_v:
        codes = codes.reshape(P, H, page // 8, 8, D).transpose(3, 4)
        scales = scales.reshape(P, H, page // 8, 8, D // 32).transpose(3, 4)
    c = codes.reshape(P, H, -1, 2)
    c = c[..., 0] | c[..., 1] << 4
    return torch.cat((c, scales.reshape(P, H, -1)), -1).reshape(P, H, page, 17 * D // 32).contiguous()


def values(cache, is_v):
    return decode(*unpack(cache, is_v))


def random_cache(g, P, H, page, D, is_v):
    """Any codes, scales near those of normal values."""
    return pack(torch.randint(0, 16, (P, H, page, D), generator=g).byte(),
                torch.randint(0x2C, 0x3E, (P, H, page, D // 32), generator=g).byte(), is_v)
