"""The operators in 8-bit floating point from their formulas in 64 bits, and how far a kernel in 32 bits may be from them.

Steps: u = 2^-24 is half a step of fp32, half of torch.finfo(t).eps that of a 16-bit type, e4m3 has half a step of 2^-4 of the
power of two below the value, and of 2^-10 below 2^-6.

* Products: an MFMA aligns the products of 8 consecutive k to the largest exponent among them, at most the exponent of the largest
  |x| of the 8 plus that of the largest |w| plus one, and cuts each at 2^-13 of it: 8 * 2^-13 times that for each eight. The 16 sums of
  a block add in fp32, each addition off by at most a step (2 u) if it truncates; kb blocks are added by FMAs (u each) with a factor of two
  roundings (the scales' product): (2 * 16 + kb + 4) u of the sum of the terms' absolute values, then the output's rounding.
* A quantized value: z = 448 v / a. v is off by dv (relative), a with it, 448 / a and the product round once each:
  z is off by 2 dv + 2 u, then half a step of e4m3 at z; the scale is off by dv + u.
* The norm: squares and sums of at most 64 values in a thread, 6 steps over lanes, 16 over waves: the sum of positive terms is off by
  at most (64 + 6 + 16 + 1) u, its root by half of that, rsqrt and division 3 u, three products 3 u: 50 u.
* silu(gate) * up: exp is off by at most 2 steps, the sum, the quotient and the product by u each, the quotient by u more where
  it is a reciprocal's: 8 u.
* The combine: one FMA a term: (topk + 1) u of the sum of absolute values, then the output's rounding.
"""
import torch

U = 2.0 ** -24
F8 = torch.float8_e4m3fn
LOW = 448 * 2.0 ** -100
NORM, SILU = 50 * U, 8 * U


def gen(dev, seed):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    return g


def half(dtype, v):
    """half a step of dtype at v"""
    if dtype == torch.float32:
        return U * v.abs() + 2.0 ** -150
    return torch.finfo(dtype).eps / 2 * (v.abs() + torch.finfo(dtype).tiny)


def within(got, want, bound, what=""):
    got, want = got.double(), want.double()
    off = (got - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} values, first at {bad.nonzero()[0].tolist()}: "
                           f"{got[bad][0].item()} for {want[bad][0].item()}, bound {torch.as_tensor(bound).expand_as(off)[bad][0].item()}")


def groups(v):
    """[t][d] -> [t][groups][128] with zeros behind"""
    t, d = v.shape
    return torch.nn.functional.pad(v, (0, -d % 128)).view(t, -(-d // 128), 128)


def check_quantized(q, s, v, dv, what=""):
    """q, s of finite values v (64 bits), which the kernel has with a relative error of at most dv"""
    t, d = v.shape
    assert q.dtype == F8 and q.shape == v.shape and s.dtype == torch.float32 and s.shape == (t, -(-d // 128)), what
    a = groups(v).abs().amax(-1).clamp_min(LOW)
    within(s, a / 448, (dv + U) * a / 448, what + " scales")
    z = (groups(v) * 448 / a[..., None]).view(t, -1)[:, :d]
    far = 2 * dv + 2 * U
    top = (z.abs() * (1 + far)).clamp_min(2.0 ** -6)
    step = torch.exp2(torch.floor(torch.log2(top)) - 4)
    within(q.float(), z, step + far * z.abs(), what + " values")


def check_16(y, v, dv, what=""):
    within(y, v, half(y.dtype, v) * (1 + dv) + dv * v.abs(), what)


def norm(h, w, eps):
    h = h.double()
    return h / (h.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()


def silu_mul(x):
    gate, up = x.double().chunk(2, 1)
    return gate * torch.sigmoid(gate) * up


def weights(dev, shape, seed):
    """e4m3 weights of all exponents and scales around 1 / 448"""
    g = gen(dev, seed)
    n, k = shape[-2:]
    q = torch.randn(*shape, device=dev, generator=g) * torch.exp2(torch.randint(-6, 7, shape, device=dev, generator=g).float())
    s = torch.exp(torch.randn(*shape[:-2], -(-n // 128), -(-k // 128), device=dev, generator=g)) / 448
    return q.clamp(-448, 448).to(F8), s


def activations(dev, t, k, seed, pad=0):
    """e4m3 rows (row stride k + pad) and scales, group-major"""
    g = gen(dev, seed)
    q = torch.randn(t, k + pad, device=dev, generator=g) * 40
    if pad:
        q[:, k:] = float("nan")  # what stands behind a row is not read as part of it
    s = torch.exp(torch.randn(-(-k // 128), t, device=dev, generator=g)) / 448
    return q.clamp(-448, 448).to(F8)[:, :k], s.t()


def _eights(v):
    """the power of two at or below the largest |v| of each 8 columns"""
    v = torch.nn.functional.pad(v.abs(), (0, -v.shape[1] % 8))
    top = v.view(v.shape[0], -1, 8).amax(-1)
    return torch.where(top > 0, torch.exp2(torch.floor(torch.log2(top.clamp_min(2.0 ** -10)))), torch.zeros_like(top))


def product(x, xs, q, s):
    """y, and how far the kernels' sums may be from it, 64 bits: one matrix"""
    n, k = q.shape
    xe, we = xs.double().repeat_interleave(128, 1), s.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)
    xd, wd = x.double() * xe[:, :k], q.double() * we[:, :k]
    off = (2 * 16 + -(-k // 128) + 4) * U * (xd.abs() @ wd.abs().t().contiguous())
    xg, wg = _eights(x.double()), _eights(q.double())
    off += 16 * 2.0 ** -13 * ((xg * xe[:, ::8][:, :xg.shape[1]]) @ (wg * we[:, ::8][:, :wg.shape[1]]).t().contiguous())
    return xd @ wd.t().contiguous(), off


def check_product(y, x, xs, q, s, what=""):
    want, off = product(x, xs, q, s)
    within(y, want, off + half(y.dtype, want.abs() + off), what)
