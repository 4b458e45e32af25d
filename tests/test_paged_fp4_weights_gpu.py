"""paged_sdpa_fp4: in how many bits the weights enter the product with the values: 22, but in fp16 calls of
tiles of 128 rows 11, unless few keys carry a row.

Half of the keys have the score 0 and the value 0, the others -6 c scale (one product, exact) and values
v, so that o = v w / (1 + w), w = exp(-6 c scale): all weights of a row but the largest are rounded alike, and an
error of w does not average out.

Bounds, u = 2^-24: the factor scale log2(e) is off by 2 u, its product with the score and exp2 by u each, so w by a relative
(3 x + 2) u, x = 6 c scale < 8; two parts of 11 bits leave 2^-22, one 2^-11 of w in the product (the sum has w itself), so of
o too; the sums of n weights and products are off by n u each, the division by 2 u; and o is rounded to fp16 once."""
import pytest
import torch

import _fp4 as F

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, F32 = torch.float16, torch.float32
I32 = torch.int32


@pytest.mark.parametrize("T", [F16, F32])
@pytest.mark.parametrize("D", [32, 64, 96, 128])
@pytest.mark.parametrize("hint", [None, 1])
def test_weights(pkg, T, D, hint):
    H, m, n, page = 4, 150, 192, 32
    k, v = torch.zeros((n, H, D)), torch.zeros((n, H, D))
    odd = torch.arange(n) % 2 == 1
    k[odd, :, 5] = -6
    v[odd] = torch.tensor([0.5, 1, 1.5, 2, 3, 4, 6, -6] * (D // 8))
    caches = []
    for x, is_v in ((k, False), (v, True)):
        codes, scales = (t.reshape(n // page, page, H, -1).transpose(1, 2).contiguous() for t in F.encode(x))
        caches.append(F.pack(codes, scales, is_v).to(DEV))
    g = torch.Generator().manual_seed(2)
    q = torch.zeros((m, H, D))
    q[..., 5] = torch.rand((m, H), generator=g) * 9 + 0.5
    q = q.to(T)
    scale = 0.140625
    i32 = lambda x: torch.tensor(x, dtype=I32, device=DEV)
    o, stats = pkg.paged_sdpa_fp4(q.to(DEV), *caches, torch.arange(n // page, dtype=I32, device=DEV)[None], i32([0, m]), i32([n]),
                                  scale=scale, causal_mask=False, max_q_len=hint)
    x = 6 * q[..., 5].double() * scale
    w = torch.exp(-x)
    ref = (w / (1 + w))[..., None] * v[1].double()
    u = 2.0 ** -24
    rel = (3 * 8.1 + 2) * u + 2.0 ** -22 + 2 * (n + 1) * u
    of_o = rel + (2.0 ** -11 if T == F16 and hint is None else 0)  # (150 rows: tiles of 128)
    # half a step at the larger of both ends
    step = torch.finfo(T).eps / 2 * 2.0 ** torch.floor(torch.log2(ref.abs() * (1 + of_o)))
    assert float(((o.double().cpu() - ref).abs() / (step + of_o * ref.abs())).max()) <= 1
    lse = torch.log(n / 2 * (1 + w))
    assert float((stats.double().cpu() - lse).abs().max()) <= rel + 8 * u * float(lse.max())
