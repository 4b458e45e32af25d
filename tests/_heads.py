"""64-bit references of the steps around attention, on the CPU, and the bounds
of their fp32 arithmetic."""
import torch

U32 = 2.0 ** -24  # half a step of fp32, relative


def half_step(t):
    """Relative bound of one rounding to t, and the absolute one of its smallest numbers."""
    fi = torch.finfo(t)
    return fi.eps / 2, fi.smallest_normal * fi.eps / 2


def tables(n, R, base=10000.0):
    freq = base ** (-torch.arange(0, R, 2, dtype=torch.float64) / max(R, 1))
    a = torch.arange(n, dtype=torch.float64)[:, None] * freq
    return a.cos().float(), a.sin().float()


def pairs(R, interleaved):
    """Indexes of the first and the second feature of every rotated pair."""
    if interleaved:
        return torch.arange(0, R, 2), torch.arange(1, R, 2)
    return torch.arange(R // 2), torch.arange(R // 2, R)


def turn(x, cos, sin, interleaved):
    """x [..., D] with its pairs turned; cos, sin [..., R / 2] broadcast against it."""
    i, j = pairs(2 * cos.shape[-1], interleaved)
    y = x.clone()
    y[..., i] = x[..., i] * cos - x[..., j] * sin
    y[..., j] = x[..., j] * cos + x[..., i] * sin
    return y


def pair_size(x, R, interleaved):
    """|x|, for rotated features the sum over their pair."""
    i, j = pairs(R, interleaved)
    y = x.abs().clone()
    y[..., i] = x[..., i].abs() + x[..., j].abs()
    y[..., j] = y[..., i]
    return y


def norm(x, w, eps):
    r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    return x * r if w is None else x * r * w


def fold(x):  # [B, S, H, D] -> [B H, S, D]
    return x.permute(0, 2, 1, 3).reshape(-1, x.shape[1], x.shape[3])


def unfold(x, B):
    return x.reshape(B, -1, x.shape[1], x.shape[2]).permute(0, 2, 1, 3)


def worst(out, ref, bound):
    """Largest error in units of its bound (a NaN counts as infinite)."""
    e = (out.detach().double().cpu() - ref).abs()
    r = torch.where(e <= bound, e / bound.clamp_min(1e-300), torch.full_like(e, float("inf")).where(e > bound, e))
    r = torch.nan_to_num(r, nan=float("inf"), posinf=float("inf"))
    return float(r.max()) if r.numel() else 0.0
