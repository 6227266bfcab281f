"""Layers in 8-bit floating point (the C-ABI's qe_rms_norm, *_f8* and qe_moe_combine entry points, include/qe_kernels.h).

8-bit values are torch.float8_e4m3fn; weights have a scale for each block of 128 x 128, activations one for each row's 128
columns. An MLP block and an expert layer, from the residual stream `h` and back:

    w1, w2 = tile_f8(q1, s1), tile_f8(q2, s2)              # once; gate and up rows in one matrix
    q, s = rms_norm(x, norm, eps, res=h, f8=True)          # h += x, then the norm of it in 8 bits
    a, t = silu_mul_f8(matmul_f8(w1, q, s))
    x = matmul_f8(w2, a, t)

    seg = moe_segment(*moe_route(logits, topk), experts, chunk)
    g = matmul_f8_grouped(w1, q, s, seg["off"], rows=seg["slot_tok"])   # w1, w2: tile_f8 of [experts][n][k]
    y = matmul_f8_grouped(w2, *silu_mul_f8(g), seg["off"])
    x = moe_combine(y, seg["inv"], weights)

Shapes, types, devices and strides are checked here (TypeError, ValueError) before the call; indexes on the device are checked
by the kernels. Calls run on the current stream of the tensors' device, need no host synchronization and can be captured.
Nothing here has a backward pass.
"""
from dataclasses import dataclass

import torch

from .attention import _run

E4M3 = torch.float8_e4m3fn
OUT_BF16, F16, W_F32 = 2, 16, 32
MAX_EXPERTS = 1024
MAX_COLS = 65536
MAX_DIM = 1 << 20
MAX_ROWS = 1 << 24
MAX_PARTS = 1 << 23
MAX_VALUES = 1 << 34
MAX_BLOCKS = 1 << 22
_OUT = {torch.float32: 0, torch.bfloat16: OUT_BF16, torch.float16: F16}
_IN = {torch.bfloat16: 0, torch.float16: F16}


# Decode loops call these wrappers for every layer and token: what is as it should be takes few reads of attributes.
def _matrix(name, t, at, align=1, far=1 << 31):
    """[rows][columns] whose rows the kernels can read: strides and place; -> row stride"""
    s = t.stride()
    if len(s) == 2 and s[1] == 1 and 0 < s[0] < far and s[0] % align == 0 and t.get_device() == at:
        return s[0]
    if t.dim() != 2:
        raise ValueError(f"{name} has two dimensions, got shape {tuple(t.shape)}")
    if t.get_device() != at:
        raise ValueError(f"{name} is on another device than the other tensors: {t.device}")
    rows, cols = t.shape
    row, col = t.stride()
    if cols > 1 and col != 1:
        raise ValueError(f"{name}: a row's values lie together, got strides {t.stride()}")
    if rows < 2:
        return -(-cols // 16) * 16  # one row: its stride may be anything
    if row >= far or row % align:
        raise ValueError(f"{name}: rows are less than {far} elements apart, by a multiple of {align}, got {row}")
    return row


def _written(name, t, shape, dtype, at):
    s = t.stride()
    if t.dtype is dtype and t.shape == shape and len(s) == 2 and s[1] == 1 and shape[1] <= s[0] < 1 << 31 and t.get_device() == at:
        return s[0]
    if t.dtype is not dtype:
        raise TypeError(f"{name} is {dtype}, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(shape)}, got {tuple(t.shape)}")
    row = _matrix(name, t, at)
    if t.shape[0] > 1 and row < t.shape[1]:
        raise ValueError(f"{name}'s rows overlap: strides {t.stride()}")
    return row


def _bytes(t):
    """bytes from a tensor's first value to the end of its last (strides are not negative)"""
    return (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()


def _apart(name, out, **others):
    """a given output shares no memory with what the call reads or writes besides (columns of one matrix are apart)"""
    a = out.data_ptr()
    for other, t in others.items():
        if t is None or not t.numel() or not out.numel():
            continue
        b = t.data_ptr()
        if b >= a + _bytes(out) or a >= b + _bytes(t):
            continue
        if out.dim() == 2 and t.dim() == 2 and out.shape[0] > 1 and t.shape[0] > 1:
            row, size, there = out.stride(0) * out.element_size(), out.shape[1] * out.element_size(), t.shape[1] * t.element_size()
            if row == t.stride(0) * t.element_size() and t.stride(1) == 1 and size <= (b - a) % row <= row - there:
                continue
        raise ValueError(f"{name} overlaps {other}")


def _same(a, b):
    return b is not None and (a is b or (a.data_ptr() == b.data_ptr() and (a.shape[0] < 2 or a.stride() == b.stride())))


def _ints(name, t, shape, at):
    if t.dtype is not torch.int32:
        raise TypeError(f"{name} is int32, got {t.dtype}")
    if t.shape != shape or not t.is_contiguous() or t.get_device() != at:
        raise ValueError(f"{name} is contiguous of shape {tuple(shape)} on {at}, got {tuple(t.shape)} on {t.device}")


def _in_type(name, t):
    f = _IN.get(t.dtype)
    if f is None:
        raise TypeError(f"{name} is bfloat16 or float16, got {t.dtype}")
    return f


def _rows_fit(t, d, what):
    if t > MAX_ROWS or d > MAX_DIM or t * -(-d // 2048) > MAX_PARTS:
        raise ValueError(f"{what}: {t} rows of {d} are too many for a call")


def _quantized(t, d, device):
    """room for [t][d] in 8 bits, rows that the products can read, and its scales, group after group"""
    q = torch.empty(t, -(-d // 16) * 16, dtype=E4M3, device=device)
    return q if d % 16 == 0 else q[:, :d], torch.empty_strided((t, -(-d // 128)), (1, t), dtype=torch.float32, device=device)


def _sizes(n, k, experts):
    if not 0 < experts <= MAX_EXPERTS or not 0 < n <= MAX_DIM or not 0 < k <= MAX_DIM or k % 16:
        raise ValueError(f"at most {MAX_EXPERTS} matrices, n and k at most {MAX_DIM}, k a multiple of 16, got {experts} of {n} x {k}")


@dataclass
class F8:
    """Weights in 8 bits (tile_f8): q uint8 in the products' layout, s fp32 [blocks of n][blocks of k], or [experts] of these."""
    q: torch.Tensor
    s: torch.Tensor
    n: int
    k: int
    experts: int = 1

    def __post_init__(self):
        _sizes(self.n, self.k, self.experts)
        blocks = (-(-self.n // 128), -(-self.k // 128))
        if self.q.dtype is not torch.uint8 or self.s.dtype is not torch.float32:
            raise TypeError(f"an F8 is uint8 with float32 scales, got {self.q.dtype} and {self.s.dtype}")
        if (self.s.shape not in (blocks, (self.experts, *blocks)) or (self.s.dim() == 2 and self.experts != 1)
                or self.q.numel() != self.experts * -(-self.n // 16) * blocks[1] * 2048 or self.q.get_device() != self.s.get_device()
                or not self.q.is_contiguous() or not self.s.is_contiguous() or self.q.data_ptr() % 16):
            raise ValueError(f"not {self.experts} matrices of {self.n} x {self.k} on one device: {tuple(self.q.shape)}, {tuple(self.s.shape)}")


def tile_f8(q, s):
    """e4m3 [n][k] with scales [ceil(n / 128)][ceil(k / 128)] fp32, or [experts][n][k] with [experts][..][..] -> F8. k is a
    multiple of 16."""
    if q.dtype is not E4M3 or s.dtype is not torch.float32:
        raise TypeError(f"weights are {E4M3} with float32 scales, got {q.dtype} and {s.dtype}")
    if q.dim() not in (2, 3):
        raise ValueError(f"weights are [n][k] or [experts][n][k], got shape {tuple(q.shape)}")
    lead, (n, k) = q.shape[:-2], q.shape[-2:]
    experts = lead[0] if lead else 1
    _sizes(n, k, experts)
    if s.shape != (*lead, -(-n // 128), -(-k // 128)):
        raise ValueError(f"scales have shape {(*lead, -(-n // 128), -(-k // 128))}, got {tuple(s.shape)}")
    at = q.get_device()
    if s.get_device() != at:
        raise ValueError(f"scales are on another device than the weights: {s.device}")
    q = q.view(-1, n, k) if q.is_contiguous() else q if lead else q[None]
    if (k > 1 and q.stride(2) != 1) or q.stride(0) % 16 and experts > 1 or q.stride(1) % 16 and n > 1 or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)
    dq = torch.empty(experts * -(-n // 16) * -(-k // 128) * 2048, dtype=torch.uint8, device=q.device)
    _run(at, "qe_tile_f8", "plliiipp", q.data_ptr(), q.stride(1) if n > 1 else k, q.stride(0) if experts > 1 else 0, n, k, experts,
         dq.data_ptr())
    return F8(dq, s.contiguous().clone(), n, k, experts)


def rms_norm(x, w, eps=1e-6, res=None, res_out=None, out=None, f8=False):
    """Root-mean-square norm of rows x [t][d] (bfloat16 or float16) with weights w [d] (their type or float32). res [t][d]: the
    residual stream; x + res, rounded to their type, goes to res_out (default: res itself; or x) and is what the norm takes.
    -> [t][d] of x's type (out, if given; x, where res_out is not); f8=True: (q, s), e4m3 with scales, and the 16-bit values go to `out` if given."""
    flags, at = _in_type("x", x), x.get_device()
    ldx = _matrix("x", x, at)
    t, d = x.shape
    if t > MAX_ROWS or not 0 < d <= MAX_COLS:
        raise ValueError(f"at most {MAX_ROWS} rows of 1 to {MAX_COLS}, got {tuple(x.shape)}")
    if not 2.0 ** -100 <= eps <= 2.0 ** 100:
        raise ValueError(f"eps is between 2^-100 and 2^100, got {eps}")
    if w.dtype is torch.float32:
        flags |= W_F32
    elif w.dtype is not x.dtype:
        raise TypeError(f"w has x's type or float32, got {w.dtype}")
    if w.shape != (d,) or not w.is_contiguous() or w.get_device() != at:
        raise ValueError(f"w is contiguous of shape {(d,)} on x's device, got {tuple(w.shape)} on {w.device}")
    ldr = ldro = 0
    if res is not None:
        if res_out is None:
            res_out = res
        ldro = _written("res_out", res_out, x.shape, x.dtype, at)
        if res.dtype is not x.dtype:
            raise TypeError(f"res is {x.dtype}, got {res.dtype}")
        if res.shape != x.shape:
            raise ValueError(f"res has x's shape {tuple(x.shape)}, got {tuple(res.shape)}")
        ldr = _matrix("res", res, at)
        to, px, pw = res_out.data_ptr(), x.data_ptr(), w.data_ptr()
        pr, rows = to if res is res_out else res.data_ptr(), 2 * (t - 1)
        end = to + rows * ldro + 2 * d
        # spans that meet are looked at closely
        if (px < end and to < px + rows * ldx + 2 * d) or (pw < end and to < pw + 4 * d) or (
                pr < end and to < pr + rows * ldr + 2 * d and (pr != to or ldr != ldro)):
            _apart("res_out", res_out, w=w, x=None if _same(res_out, x) else x, res=None if _same(res_out, res) else res)
    elif res_out is not None:
        raise ValueError("res_out without res")
    y, ldy, q, s = out, 0, None, None
    if out is not None:
        ldy = _written("out", out, x.shape, x.dtype, at)
        _apart("out", out, w=w, x=None if _same(out, x) else x, res=res, res_out=res_out)
    elif not f8:
        y = torch.empty(t, d, dtype=x.dtype, device=x.device)
        ldy = d
    if f8:
        q, s = _quantized(t, d, x.device)
    if t:
        _run(at, "qe_rms_norm", "plplplpfplplplliiip", x.data_ptr(), ldx, None if res is None else res.data_ptr(), ldr,
             None if res is None else res_out.data_ptr(), ldro, w.data_ptr(), eps, None if y is None else y.data_ptr(), ldy,
             q.data_ptr() if f8 else None, q.stride(0) if f8 else 0, s.data_ptr() if f8 else None, 1, t, t, d, flags)
    return (q, s) if f8 else y


def _act(x, glu):
    flags, at = _in_type("x", x), x.get_device()
    ldx = _matrix("x", x, at)
    t, d = x.shape
    if glu:
        if d % 2:
            raise ValueError(f"rows hold as many gate as up values, got {d}")
        d //= 2
    _rows_fit(t, d, "x")
    if d == 0:
        raise ValueError("rows without columns")
    q, s = _quantized(t, d, x.device)
    if t:
        _run(at, "qe_act_f8", "pliplplliiip", x.data_ptr(), ldx, int(glu), q.data_ptr(), q.stride(0), s.data_ptr(), 1, t, t, d, flags)
    return q, s


def quant_f8(x):
    """rows x [t][d] (bfloat16 or float16) in 8 bits -> (q e4m3 [t][d], s fp32 [t][ceil(d / 128)])"""
    return _act(x, False)


def silu_mul_f8(x):
    """silu(gate) * up of rows x [t][2 d] = [gate][up] (bfloat16 or float16), in 8 bits -> (q [t][d], s [t][ceil(d / 128)])"""
    return _act(x, True)


def _operands(w, q, s, experts):
    if not isinstance(w, F8):
        raise TypeError(f"weights are an F8, got {type(w).__name__}")
    if q.dtype is not E4M3 or s.dtype is not torch.float32:
        raise TypeError(f"activations are {E4M3} with float32 scales, got {q.dtype} and {s.dtype}")
    at = w.q.get_device()
    if experts != (w.s.dim() == 3):
        raise ValueError("one matrix for matmul_f8, [experts] of them for matmul_f8_grouped")
    ldx = _matrix("q", q, at, 16, 1 << 24)
    t = q.shape[0]
    if q.shape[1] != w.k or t > MAX_ROWS:
        raise ValueError(f"q is at most {MAX_ROWS} rows of {w.k}, got {tuple(q.shape)}")
    if q.data_ptr() % 16:
        raise ValueError("q is 16-byte aligned")
    if s.shape != (t, -(-w.k // 128)) or s.get_device() != at:
        raise ValueError(f"scales have shape {(t, -(-w.k // 128))} on the weights' device, got {tuple(s.shape)} on {s.device}")
    if t > 1 and s.stride(0) >= 1 << 22:
        raise ValueError(f"scales of rows are less than 2^22 elements apart, got {s.stride(0)}")
    return at, ldx, t


def _product(w, r, dtype, y, at, blocks=0):
    dtype = dtype if y is None else y.dtype
    flags = _IN.get(dtype)
    if flags is None:
        raise TypeError(f"products are bfloat16 or float16, got {dtype}")
    if r > MAX_ROWS or r * w.n > MAX_VALUES or blocks > MAX_BLOCKS:
        raise ValueError(f"{r} rows of {w.n} are too many for a call")
    if y is None:
        y = torch.empty(r, w.n, dtype=dtype, device=w.q.device)
        return y, w.n, flags
    return y, _written("y", y, (r, w.n), y.dtype, at), flags


def matmul_f8(w: F8, q, s, dtype=torch.bfloat16, y=None):
    """y [t][n] = rows (q e4m3 [t][k], s fp32 [t][ceil(k / 128)]) times the matrix w; into y, or a new tensor of
    type dtype (bfloat16 or float16)"""
    at, ldx, t = _operands(w, q, s, False)
    given = y is not None
    y, ldy, flags = _product(w, t, dtype, y, at)
    if given:
        _apart("y", y, q=q, s=s, weights=w.q, scales=w.s)
    if t:
        _run(at, "qe_matmul_f8", "ppiiplplliplip", w.q.data_ptr(), w.s.data_ptr(), w.n, w.k, q.data_ptr(), ldx, s.data_ptr(), s.stride(0),
             s.stride(1), t, y.data_ptr(), ldy, flags)
    return y


def matmul_f8_choice(w: F8, q, s, bt, bw, parts, dtype=torch.bfloat16):
    """matmul_f8 by a given kernel and number of K ranges instead of those that its sizes choose (qe_matmul_f8_choice)"""
    at, ldx, t = _operands(w, q, s, False)
    if not (bt == 16 or (bt == bw == 256) or (bt in (32, 64, 128) and bw in (64, 128, 192))) or not 1 <= parts <= min(16, -(-w.k // 128)):
        raise ValueError(f"no blocks of {bt} x {bw} with {parts} K ranges")
    if -(-t // bt) * -(-w.n // (32 if bt == 16 else bw)) * parts > MAX_BLOCKS or not t:
        raise ValueError(f"{t} rows of {w.n} in {parts} ranges")
    y, ldy, flags = _product(w, t, dtype, None, at)
    _run(at, "qe_matmul_f8_choice", "ppiiplpllipliiiip", w.q.data_ptr(), w.s.data_ptr(), w.n, w.k, q.data_ptr(), ldx, s.data_ptr(), s.stride(0),
         s.stride(1), t, y.data_ptr(), ldy, flags, bt, bw, parts)
    return y


def matmul_f8_grouped(w: F8, q, s, off, rows=None, dtype=torch.bfloat16, y=None):
    """Rows off[e] .. off[e + 1] - 1 of y (off int32 [experts + 1], ascending) = matrix e of w times the same rows of (q, s), or
    rows[i] of them for row i (rows int32; a number outside q gives a row of zeros). Rows of y in no segment are left as
    they were in a given y (and have no meaning in a new one). y has as many rows as `rows`, or as q."""
    at, ldx, t = _operands(w, q, s, True)
    _ints("off", off, (w.experts + 1,), at)
    r = t
    if rows is not None:
        _ints("rows", rows, (rows.numel(),), at)
        r = rows.numel()
    given = y is not None
    rows_a_block, cols = (16, 32) if r // w.experts < 8 else (64, 128)  # the smallest blocks that the library may take
    y, ldy, flags = _product(w, r, dtype, y, at, (r // rows_a_block + min(r, w.experts)) * -(-w.n // cols))
    if given:
        _apart("y", y, q=q, s=s, weights=w.q, scales=w.s, off=off, rows=rows)
    if r:
        _run(at, "qe_matmul_f8_grouped", "ppiiiplpllippiplip", w.q.data_ptr(), w.s.data_ptr(), w.n, w.k, w.experts, q.data_ptr(), ldx,
             s.data_ptr(), s.stride(0), s.stride(1), t, off.data_ptr(), None if rows is None else rows.data_ptr(), r, y.data_ptr(), ldy, flags)
    return y


def matmul_f8_grouped_choice(w: F8, q, s, off, bt, rows=None, dtype=torch.bfloat16, y=None):
    """matmul_f8_grouped by a given kernel instead of the one that its sizes choose (qe_matmul_f8_grouped_choice)"""
    at, ldx, t = _operands(w, q, s, True)
    _ints("off", off, (w.experts + 1,), at)
    if rows is not None:
        _ints("rows", rows, (rows.numel(),), at)
    r = t if rows is None else rows.numel()
    if bt not in (16, 64, 128, 256) or (bt == 256 and rows is not None and t * max(ldx, s.stride(0) * 4) >= 1 << 32) or not r:
        raise ValueError(f"no blocks of {bt} for {r} of {t} rows")
    given = y is not None
    y, ldy, flags = _product(w, r, dtype, y, at, (r // bt + min(r, w.experts)) * -(-w.n // {16: 32, 256: 256}.get(bt, 128)))
    if given:
        _apart("y", y, q=q, s=s, weights=w.q, scales=w.s, off=off, rows=rows)
    _run(at, "qe_matmul_f8_grouped_choice", "ppiiiplpllippipliip", w.q.data_ptr(), w.s.data_ptr(), w.n, w.k, w.experts, q.data_ptr(), ldx,
         s.data_ptr(), s.stride(0), s.stride(1), t, off.data_ptr(), None if rows is None else rows.data_ptr(), r, y.data_ptr(), ldy, flags, bt)
    return y


def moe_combine(y, inv, w, add=None, out=None):
    """out [t][d] = add + sum over j of w[i][j] * y[inv[i * topk + j]]: the rows y [slots][d] of a grouped product back into
    tokens, inv int32 [t * topk] and w fp32 [t][topk] as moe_segment and moe_route give them (an index outside y adds nothing).
    y: bfloat16, float16 or float32; out (default: new, of add's or y's type; it may be add itself) and add have y's type or
    float32."""
    yflags, at = _OUT.get(y.dtype), y.get_device()
    if yflags is None:
        raise TypeError(f"y is bfloat16, float16 or float32, got {y.dtype}")
    ldy = _matrix("y", y, at)
    if w.dtype is not torch.float32:
        raise TypeError(f"w is float32, got {w.dtype}")
    if w.dim() != 2 or not w.is_contiguous() or w.get_device() != at:
        raise ValueError(f"w is contiguous [t][topk] on y's device, got {tuple(w.shape)} on {w.device}")
    (t, topk), (slots, d) = w.shape, y.shape
    _ints("inv", inv, (t * topk,), at)
    _rows_fit(t, d, "y")
    if slots >= 1 << 31 or topk > 1024 or d == 0:
        raise ValueError(f"at most 2^31 rows and 1024 of them a token, got {tuple(y.shape)} and {tuple(w.shape)}")
    dtype = out.dtype if out is not None else add.dtype if add is not None else y.dtype
    if dtype not in (y.dtype, torch.float32):
        raise TypeError(f"out and add have y's type or float32, got {dtype}")
    ldadd = 0 if add is None else _written("add", add, (t, d), dtype, at)
    if out is None:
        out = torch.empty(t, d, dtype=dtype, device=y.device)
        ldout = d
    else:
        ldout = _written("out", out, (t, d), dtype, at)
        _apart("out", out, y=y, inv=inv, w=w, add=None if _same(out, add) else add)
    if t:
        _run(at, "qe_moe_combine", "plippplpliiiiip", y.data_ptr(), ldy, slots, inv.data_ptr(), w.data_ptr(),
             None if add is None else add.data_ptr(), ldadd, out.data_ptr(), ldout, t, topk, d, yflags, _OUT[dtype])
    return out
