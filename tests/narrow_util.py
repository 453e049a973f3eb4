"""Plain 64-bit forms of the layers of narrow types, and what their tests share."""
import torch

from smallframework_b200 import interface as S

F8 = torch.float8_e4m3fn
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BUFFERS = {torch.float32: S.FloatBuffer, torch.bfloat16: S.BFloat16Buffer, torch.float16: S.HalfBuffer}


def buffer(t):
    return BUFFERS[t.dtype](data=t)


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def cdiv(a, b):
    return -(-a // b)


def spread(scales, rows, columns, block_rows):
    s = scales.view(-1, cdiv(columns, 128)).double()
    return s.repeat_interleave(block_rows, 0)[:rows].repeat_interleave(128, 1)[:, :columns]


def quantize(x, block_rows):
    """Codes (as doubles) and scales of a matrix of finite values, by the definition: every e4m3 value in a table, the nearest found by its middles."""
    rows, columns = x.shape
    r, c = cdiv(rows, block_rows), cdiv(columns, 128)
    whole = torch.zeros(r * block_rows, c * 128, dtype=torch.float64, device=x.device)
    whole[:rows, :columns] = x.double()
    amax = whole.abs().view(r, block_rows, c, 128).amax((1, 3)).float()
    scales = torch.where(amax > 0, (amax / torch.full_like(amax, 448)).clamp_min(2.0 ** -126), torch.ones_like(amax))
    table = torch.tensor([m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)][:-1],
                         dtype=torch.float64, device=x.device)
    middle = (table[1:] + table[:-1]) / 2
    q = x.double() / spread(scales, rows, columns, block_rows)
    below, above = torch.searchsorted(middle, q.abs()), torch.searchsorted(middle, q.abs(), right=True)
    return torch.copysign(table[torch.where(below % 2 == 0, below, above)], q), scales


def operand(rows, columns, block_rows, seed, spread_of_scales=2.0):
    """A Float8Buffer of random codes (no NaN) and scales of many magnitudes."""
    g = generator(seed)
    codes = torch.randn(rows, columns, generator=g, device="cuda").mul(60).clamp(-448, 448).to(F8)
    n = cdiv(rows, block_rows) * cdiv(columns, 128)
    scales = torch.exp(torch.randn(n, generator=g, device="cuda") * spread_of_scales) * 1e-2
    return S.Float8Buffer(rows, columns, block_rows, data=codes, scales=scales)


def values(b):
    return b.t.view(b.rows, b.columns).double() * spread(b.scales, b.rows, b.columns, b.block_rows)


def dense(x, w, bias=None, act=0, slope=0.0, before=None):
    """The layer in 64 bits, and the sum of magnitudes that its roundings are relative to."""
    xv, wv = values(x), values(w)
    size = xv.abs() @ wv.abs().t()
    y = torch.zeros_like(size)
    for b in range(cdiv(x.columns, 128)):  # a block's sum and then its scales, as the layer is defined: an infinite scale of a sum is one
        at = slice(128 * b, 128 * b + 128)
        sw = w.scales.view(-1, cdiv(w.columns, 128))[:, b].double().repeat_interleave(128)[:w.rows]
        y += (x.t.view(x.rows, -1)[:, at].double() @ w.t.view(w.rows, -1)[:, at].double().t()) * (x.scales.view(x.rows, -1)[:, b].double()[:, None] * sw)
    if before is not None:
        y, size = y + before.double(), size + before.double().abs()
    if bias is not None:
        y, size = y + bias.double(), size + bias.double().abs()
    if act:
        y = torch.where(y > 0, y, y * (slope if act == 2 else 0.0))
    return y, size


def dense_tolerance(y, size, inputs, kind):
    """Products of e4m3 numbers are exact in fp32.  A block's 128 are added with at most one truncation (2^-23) each, the two scales' product is
    one rounding (2^-24), and every block, the old value and the bias one more; at the end the rounding to the output's type."""
    eps = 128 * 2.0 ** -23 + (cdiv(inputs, 128) + 3) * 2.0 ** -24
    out = torch.finfo(kind).eps / 2
    return size * eps * (1 + out) + y.abs() * out + torch.finfo(kind).tiny


def overflows(got, want, tolerance, kind):
    """Infinities of a result where the type has them: beyond its largest value by half a step or more, after at most `tolerance`."""
    last = torch.finfo(kind).max * (1 + torch.finfo(kind).eps / 4)
    return got.isinf() & (torch.sign(got.double()) == torch.sign(want)) & (want.abs() + tolerance >= last)


def logprobs(x, tokens, top):
    x = x.double()
    m = x.amax(1, keepdim=True)
    nothing = (x == -torch.inf).all(1, keepdim=True)
    t = x - torch.where(nothing, 0.0, m)  # first: beside a mask of the type's lowest value a logarithm would be lost
    z = torch.where(nothing, 1.0, t.exp().sum(1, keepdim=True)).log()
    logp = t - z
    p = logp.exp()
    h = -torch.where(p == 0, 0.0, p * logp).sum(1)
    given = logp.gather(1, tokens.clamp(0, x.shape[1] - 1)[:, None]).squeeze(1)
    given = torch.where(tokens < 0, 0.0, torch.where(tokens >= x.shape[1], torch.nan, given))
    rank = torch.where(x.isnan(), -torch.inf, x)
    best = torch.sort(rank, dim=1, descending=True, stable=True).indices[:, :top]
    return given, h, torch.where(z.isnan(), torch.nan, logp.gather(1, best)), best
