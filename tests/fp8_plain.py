"""8-bit floating point in plain form: how blocks are held (32-bit operations, as they are defined) and products in 64 bits."""
import torch

B, F8 = 128, torch.float8_e4m3fn
EPS = 2.0 ** -24                                 # half a step of a 32-bit value of one


def blocks_of(n):
    return -(-n // B)


def held(x):
    """(q float8 [T, blocks * 128], scale float32 [blocks, T]) of x [T, K]."""
    t, k = x.shape
    full = torch.zeros(t, blocks_of(k) * B, dtype=torch.float32, device=x.device)
    full[:, :k] = x.float()
    blocks = full.view(t, -1, B)
    m = blocks.abs().amax(-1).clamp_min(2.0 ** -100)
    most = torch.full_like(m, 448.0)
    q = (blocks * (most / m)[..., None]).to(F8).view(t, -1)
    return q, (m / most).t().contiguous()


def held_matrix(w):
    """(q [N, blocks * 128], scale [ceil(N / 128), blocks]) of a matrix."""
    n, k = w.shape
    nb, kb = blocks_of(n), blocks_of(k)
    full = torch.zeros(nb * B, kb * B, dtype=torch.float32, device=w.device)
    full[:n, :k] = w.float()
    tiles = full.view(nb, B, kb, B)
    m = tiles.abs().amax((1, 3)).clamp_min(2.0 ** -100)
    most = torch.full_like(m, 448.0)
    q = (tiles * (most / m)[:, None, :, None]).view(nb * B, kb * B)[:n].to(F8)
    return q, m / most


def rows_values(q, scale):
    return (q.double().view(q.shape[0], -1, B) * scale.t().double()[:, :, None]).flatten(1)


def matrix_values(q, scale):
    n = q.shape[0]
    at = torch.arange(n, device=q.device) // B
    return (q.double().view(n, -1, B) * scale.double()[at][:, :, None]).flatten(1)


def gate_up_values(q, scale):
    n = q.shape[0] // 2
    both = q.view(n // 8, 2, 8, -1)
    return [matrix_values(both[:, i].reshape(n, -1), scale[i]) for i in (0, 1)]


def random_matrix(n, k, device, seed, stack=None, gated=False):
    """(q, scale) of a random matrix; gated: 2 n rows in eights."""
    g = torch.Generator(device=device).manual_seed(seed)
    lead, rows, sets = ((stack,) if stack else ()), (2 * n if gated else n), ((2,) if gated else ())
    v = 100 * torch.randn(*lead, rows, blocks_of(k) * B, generator=g, device=device)
    v[..., k:] = 0
    scale = 1e-3 * torch.exp(torch.randn(*lead, *sets, blocks_of(n), blocks_of(k), generator=g, device=device))
    return v.clamp(-448, 448).to(F8), scale


def sum_bound(blocks):
    """Error of a product's 32-bit sums, in parts of the sum of the products' sizes.  A tensor-core instruction adds 32 products (exact: 4 + 4 bits) to
    what it has, each of the 33 cut at no less than the 24th bit of the largest: 33 * 2^-23, four instructions a block.  The two scales' product, its
    product with the block's sum and the sum over blocks are rounded to 32 bits: blocks + 2 roundings of 2^-24."""
    return 4 * 33 * 2 * EPS + (blocks + 2) * EPS
