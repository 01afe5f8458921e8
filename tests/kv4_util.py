"""The 4-bit cache's numbers in 64 bits, apart from the kernels: what is held
for a row, what a cache's bytes stand for."""
import torch

MAGNITUDES = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
# every scale: m / 8 * 2^-14 below 2^-14, (1 + m / 8) * 2^(e - 15) from there
SCALES = torch.tensor([(e * 8 + m) * 2.0 ** -17 if e == 0 else (8 + m) * 2.0 ** (e - 18) for e in range(31) for m in range(8)],
                      dtype=torch.float64)
TOP = 61440.0  # six of the largest scale a row takes, 10240


def quantised(x):
    """Codes (0 to 15), bytes of scales and values of rows x [..., dim]."""
    x = x.cpu().double()
    x = torch.where(torch.isnan(x), TOP, x).clamp(-TOP, TOP)
    d = x.shape[-1]
    x = torch.nn.functional.pad(x, (0, -d % 32)).unflatten(-1, (-1, 32))
    byte = torch.searchsorted(SCALES * 6, x.abs().amax(-1).contiguous())
    scale = SCALES[byte][..., None]
    r = torch.where(scale > 0, x.abs() / scale, 0)[..., None]  # (a border of two numbers is one exactly)
    off = (r - MAGNITUDES).abs()
    # the nearest, of two as near the even code
    code = (off * 2 + 1e-9 * (torch.arange(8) % 2)).argmin(-1)
    value = MAGNITUDES[code] * scale * torch.where(x < 0, -1.0, 1.0)
    code = code + 8 * (x < 0)
    return code.flatten(-2)[..., :d], byte, value.flatten(-2)[..., :d]


def numbers(cache, name):
    """What a cache's K or V holds, [blocks * block, heads, dim] in 64 bits."""
    codes, scale = getattr(cache, name).cpu().long(), getattr(cache, name + "_scale").cpu().long()
    n, h, _, block = scale.shape
    four = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    if name == "v":
        four = four.transpose(-1, -2).reshape(n, h, block, -1)
    s = torch.cat([SCALES, torch.full((8,), float("nan"), dtype=torch.float64)])[scale]
    x = MAGNITUDES[four & 7] * torch.where(four > 7, -1.0, 1.0) * s.transpose(2, 3).repeat_interleave(32, -1)
    return x.transpose(1, 2).flatten(0, 1)[..., :cache.head_dim]
