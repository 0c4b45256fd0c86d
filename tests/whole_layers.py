"""Row-wise layers of whole numbers: every sum of products is one below 2^24, exact in 32 bits in whatever order, so that a result is
that of the formula rounded once, bit for bit, and a row that is lost or counted twice is seen."""
import torch

# rows, channels in and out: few channels in several rounds of every workgroup; every tile in every layout, whole and in slices
NARROW = [(32773, 24, 48), (70000, 128, 128), (70001, 64, 128), (33000, 128, 40), (119985, 64, 64)]
LARGE = [(4093, 1000, 4088), (4093, 4088, 1000), (66000, 264, 680), (65272, 680, 168), (8200, 2040, 1030), (20000, 512, 520), (700, 20000, 500), (42200, 392, 568)]
# rows and their length
NORMS = [(70001, 64), (60000, 128), (30000, 500), (20000, 1024), (8191, 2048), (5000, 4096), (3000, 8192), (2000, 16384), (700, 20000), (300, 40000)]


def whole(g, most, *shape):
    return torch.randint(-most, most + 1, shape, generator=g, device=g.device, dtype=torch.int8)


def linear(m, k, n, device):
    """x, weight, bias, residual, gradient of the result: small whole numbers (few in a weight's row, so that results are exact too)"""
    g = torch.Generator(device=device).manual_seed(m + k)
    w = whole(g, 1, n, k) * (torch.rand(n, k, generator=g, device=device) < 24 / k)
    return whole(g, 2, m, k), w, whole(g, 2, n), whole(g, 3, m, n), whole(g, 2, m, n)


def linear_want(x, w, b, r, dy, relu):
    """z, the result, and dz, in 32 bits"""
    z = torch.mm(x.float(), w.float().t().contiguous()) + b.float()
    dz = torch.where(z > 0, dy.float(), 0.0) if relu else dy.float()
    return z, (z.clamp_min(0) if relu else z) + r.float(), dz


def norm(m, k, device):
    """x of +-2, gradients of the result and of the sum"""
    g = torch.Generator(device=device).manual_seed(m + k)
    signs = 2 * whole(g, 1, m, k).ne(0).to(torch.int8) - 1
    return 2 * signs, whole(g, 2, m, k), whole(g, 2, m, k)
