"""MXFP4 blocks and the pages of a cache that holds them, from the format's
definition (include/tbq_kv.h), on the CPU in 64 bits: values to codes and scale
bytes, and pages of bytes to values and back."""
import torch

GRID = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
LEAST, MOST, NAN = -23, 13, 255


def blocks(x):
    """(codes [..., D], scale bytes [..., D / 32]) of rows x [..., D] (64 bits)."""
    b = x.double().unflatten(-1, (-1, 32))
    odd = ~torch.isfinite(b).all(-1)
    b = torch.where(odd[..., None], torch.zeros(()).double(), b)
    a = b.abs().amax(-1)
    E = torch.full(a.shape, LEAST)
    for e in range(LEAST, MOST):
        E = E + (a > 7 * 2.0 ** e)
    y = b / (2.0 ** E.double())[..., None]
    d = (y.abs()[..., None] - GRID).abs()
    near = d == d.amin(-1, keepdim=True)
    # of two codes that are equally near, the even one
    code = (near & (torch.arange(8) % 2 == 0)).double().argmax(-1)
    code = torch.where((near & (torch.arange(8) % 2 == 0)).any(-1), code, near.double().argmax(-1))
    code = code + 8 * torch.signbit(y)
    return code.flatten(-2), torch.where(odd, NAN, E + 127)


def unblock(code, scale):
    v = torch.where(code >= 8, -1.0, 1.0).double() * GRID[code % 8]
    s = torch.where(scale == NAN, float("nan"), 2.0 ** (scale.double() - 127))
    return (v.unflatten(-1, (-1, 32)) * s[..., None]).flatten(-2)


def rounded(x):
    """What the cache gives back for rows x."""
    return unblock(*blocks(x))


def places(page, D, is_v):
    """Byte of every element [page][D], and byte of every scale [page][D / 32], of a kv head's page."""
    r, d, b = torch.arange(page)[:, None], torch.arange(D)[None], torch.arange(D // 32)[None]
    end = page * D // 2
    if is_v:
        return ((r // 4 * (D // 8) + d // 8) * 4 + r % 4) * 4 + d % 8 // 2, end + (r // 4 * (D // 32) + b) * 4 + r % 4
    return r * (D // 2) + d // 2, end + r * (D // 32) + b


def pack(code, scale, is_v):
    """Pages [..., bytes] (uint8) of codes [..., page, D] and scale bytes [..., page, D / 32]."""
    page, D = code.shape[-2:]
    at, sc = places(page, D, is_v)
    out = torch.zeros(code.shape[:-2] + (page * (D // 2 + D // 32),), dtype=torch.uint8)
    c = code.to(torch.uint8)
    out[..., at[:, 0::2].flatten()] = (c[..., 0::2] | c[..., 1::2] << 4).flatten(-2)
    out[..., sc.flatten()] = scale.to(torch.uint8).flatten(-2)
    return out


def unpack(pages, page, D, is_v):
    """(codes, scale bytes) of pages [..., bytes]."""
    at, sc = places(page, D, is_v)
    b = pages[..., at.flatten()].unflatten(-1, (page, D)).long()
    return torch.where(torch.arange(D) % 2 == 1, b >> 4, b & 15), pages[..., sc.flatten()].unflatten(-1, (page, D // 32)).long()


def values(pages, page, D, is_v):
    """Values [..., page, D] (64 bits) that pages [..., bytes] hold."""
    return unblock(*unpack(pages, page, D, is_v))


def pool(x, is_v):
    """Pages of the rows x [..., page, D]."""
    return pack(*blocks(x), is_v)
