"""Rows, products, cache and attention in 8-bit codes, against their definitions in 64 bits.

A row x is codes c and a scale s = max|x| / 127; c = x / s rounded to the nearest integer, halves to the even one.
"""
import math

import pytest
import torch

from kvad_b200.ops import KernelError, Ops

pytestmark = pytest.mark.gpu
DT = {"float32": torch.float32, "bfloat16": torch.bfloat16}
U = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8}         # a rounding's relative size
PAGE = 64


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def held(x):
    """Codes and scales of rows (the last axis), in x's own precision."""
    s = x.abs().amax(-1) * x.new_tensor(1 / 127)
    return torch.round(x / torch.where(s > 0, s, 1).unsqueeze(-1)).clamp(-127, 127), s


def apart(t, extra=3):
    """The same numbers as columns of a wider buffer (rows that lie apart, and not on 16-byte boundaries where `extra` is odd)."""
    wide = torch.full((t.shape[0], t.shape[1] + extra), 77, dtype=t.dtype, device=t.device)
    wide[:, :t.shape[1]] = t
    return wide[:, :t.shape[1]]


# -- rows ---------------------------------------------------------------------------------------------------------------------


# a warp's rows and a block's, widths that end inside a thread's four entries, the widest; rows that lie together and apart
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("n,width", [(1, 1), (5, 3), (9, 64), (130, 128), (7, 130), (33, 512), (3, 516), (2, 1600), (5, 2049), (3, 4100), (2, 9000), (1, 16400), (2, 32768)])
@pytest.mark.parametrize("extra", [0, 3, 16])
def test_rows_become_the_codes_of_the_definition(dtype, n, width, extra):
    x = torch.randn(n, width, device="cuda", generator=generator(width + n)).to(DT[dtype])
    x[0, 0] *= 50
    if n > 2:
        x[1] = 0
        x[2] *= 1e-44 / x[2].abs().max().float() if dtype == "float32" else 1e-30
    src = apart(x, extra) if extra else x
    codes = apart(torch.zeros(n, width, dtype=torch.int8, device="cuda"), extra) if extra else torch.zeros(n, width, dtype=torch.int8, device="cuda")
    scales = torch.full((n,), -1.0, device="cuda")
    Ops(DT[dtype]).int8_rows(src, codes, scales)
    want, s = held(x.float())
    assert torch.equal(scales, s)
    assert torch.equal(codes.float(), want)
    for out_dtype in DT.values():
        out = apart(torch.zeros(n, width, dtype=out_dtype, device="cuda"), extra) if extra else torch.zeros(n, width, dtype=out_dtype, device="cuda")
        Ops(DT[dtype]).int8_read(codes, scales, out)
        assert torch.equal(out, (want * s.unsqueeze(1)).to(out_dtype))
    # each entry is within half a scale of what it stands for (and a rounding of the quotient, and of the product)
    if n <= 2:
        off = ((codes.double() * scales.double().unsqueeze(1)) - x.double()).abs()
        assert (off <= scales.double().unsqueeze(1) * (0.5 + 127 * 2.0 ** -22)).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("width", [48, 700])
def test_a_row_that_is_not_finite_says_so_and_leaves_the_others_alone(bad, width):
    x = torch.randn(6, width, device="cuda", generator=generator(1))
    want, s = held(x)
    x[2, width - 1] = bad
    codes, scales = torch.empty(6, width, dtype=torch.int8, device="cuda"), torch.empty(6, device="cuda")
    Ops(torch.bfloat16).int8_rows(x, codes, scales)
    assert scales[2].isnan() and (codes[2] == 0).all()
    others = [0, 1, 3, 4, 5]
    assert torch.equal(codes[others].float(), want[others]) and torch.equal(scales[others], s[others])


@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("n,width,extra", [(1, 16, 0), (8, 1024, 0), (3, 1600, 0), (5, 257, 0), (4, 300, 3), (9, 77, 1), (2, 6400, 8), (1, 20000, 0), (149, 700, 0), (150, 1500, 0), (149, 2048, 0), (151, 3000, 0), (149, 4096, 0), (149, 6000, 0), (149, 8192, 0),
                                           (149, 16000, 0), (2, 4096, 0), (2, 8000, 0)])
@pytest.mark.parametrize("params", ["float32", "bfloat16", None])
@pytest.mark.parametrize("delta", [None, "float32", "bfloat16"])
def test_normed_rows(norm, n, width, extra, params, delta):
    g = generator(n * width)
    x = torch.randn(n, width, device="cuda", generator=g) * 3 + 0.5
    w = None if params is None else (1 + 0.1 * torch.randn(width, device="cuda", generator=g)).to(DT[params])
    b = None if params is None or norm == "rms" else (0.1 * torch.randn(width, device="cuda", generator=g)).to(DT[params])
    d = None if delta is None else torch.randn(n, width, device="cuda", generator=g).to(DT[delta])
    mult, eps, unit = 0.75, 1e-5, norm == "rms" and params is not None
    t = x.double() if d is None else x.double() + mult * d.double()
    y = t - t.mean(-1, keepdim=True) if norm == "layer" else t
    y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps)
    if w is not None:
        y = y * (w.double() + (1 if unit else 0))
    if b is not None:
        y = y + b.double()
    put = (lambda z: apart(z, extra)) if extra else (lambda z: z)
    ops = Ops(torch.bfloat16)
    stream, codes, scales = put(x.clone()), put(torch.zeros(n, width, dtype=torch.int8, device="cuda")), torch.zeros(n, device="cuda")
    aside = None if n % 2 else put(torch.zeros(n, width, device="cuda"))        # the sum goes to a buffer of its own, or into the stream
    more = {"delta": None if d is None else put(d), "mult": mult, "x_out": aside}
    if norm == "rms":
        ops.rmsnorm_int8(stream, w, eps, codes, scales, unit_offset=unit, **more)
    else:
        ops.layernorm_int8(stream, w, b, eps, codes, scales, **more)
    if aside is not None:
        assert torch.equal(stream, x)
        assert ((aside.double() - t).abs() <= 2.0 ** -23 * t.abs().clamp_min(1)).all()
    else:
        assert ((stream.double() - t).abs() <= 2.0 ** -23 * t.abs().clamp_min(1)).all()
    # a thread's chain of at most 32 terms and a tree of 10 in the mean square (halved by the root) and in the mean (of numbers up to 15), then some ten roundings
    size = y.abs().amax(-1)
    off = (32 + 10 + 12) * 2.0 ** -24 * (1 + (4 if norm == "layer" else 0)) * size + 2.0 ** -23
    assert ((scales.double() - size / 127).abs() <= off / 127 + 2.0 ** -23 * size / 127).all()
    assert ((codes.double() * scales.double().unsqueeze(1) - y).abs() <= (scales.double() * 0.5 + 2 * off).unsqueeze(1)).all()


def test_normed_rows_of_a_list():
    x = torch.randn(20, 640, device="cuda", generator=generator(3))
    w = 1 + 0.1 * torch.randn(640, device="cuda", generator=generator(4))
    rows = torch.tensor([19, 0, 7], dtype=torch.int32, device="cuda")
    ops = Ops(torch.float32)
    all_codes, all_scales = torch.empty(20, 640, dtype=torch.int8, device="cuda"), torch.empty(20, device="cuda")
    codes, scales = torch.empty(3, 640, dtype=torch.int8, device="cuda"), torch.empty(3, device="cuda")
    ops.rmsnorm_int8(x, w, 1e-6, all_codes, all_scales)
    ops.rmsnorm_int8(x, w, 1e-6, codes, scales, rows=rows)
    assert torch.equal(codes, all_codes[rows.long()]) and torch.equal(scales, all_scales[rows.long()])


# -- products -----------------------------------------------------------------------------------------------------------------


def product(seed, m, n, k, extra=0):
    g = generator(seed)
    a = torch.randint(-127, 128, (m, k), dtype=torch.int8, device="cuda", generator=g)
    w = torch.randint(-127, 128, (n, k), dtype=torch.int8, device="cuda", generator=g)
    sa = torch.rand(m, device="cuda", generator=g) * 0.02 + 1e-3
    sw = torch.rand(n, device="cuda", generator=g) * 0.02 / math.sqrt(k) + 1e-5
    return (apart(a, extra) if extra else a), sa, w, sw, torch.randn(n, device="cuda", generator=g)


def gelu(y, form):
    if form == "gelu_erf":
        return y * 0.5 * torch.erfc(-y / math.sqrt(2))
    return y / (1 + torch.exp(-2 * 0.79788456 * (y + 0.044715 * y ** 3)))


def check_product(dtype, m, n, k, epilogue, bias=True, extra=0, form=0):
    a, sa, w, sw, b = product(m + n + k, m, n, k, extra)
    b = b if bias is True else None if not bias else b.to(DT[bias])
    whole = (a.double() @ w.double().T)                      # exact: every sum is below 2^53
    y = whole * sa.double().unsqueeze(1) * sw.double() + (0 if b is None else b.double())
    out_dtype = torch.float32 if epilogue in ("residual", "store_f32") else DT[dtype]
    base = torch.randn(m, n, device="cuda", generator=generator(5)) if epilogue == "residual" else torch.full((m, n), float("nan"), device="cuda")
    out = apart(base.to(out_dtype), 5) if extra else base.to(out_dtype).clone()
    Ops(DT[dtype]).linear_int8(a, sa, w, sw, b, out, epilogue, form=form)
    # the sum's own rounding to 32 bits, the two scales', the bias'
    off = 4 * 2.0 ** -24 * ((y - (0 if b is None else b.double())).abs() + y.abs())
    if epilogue == "residual":
        y = y + base.double()
        off = off + 2.0 ** -24 * y.abs()
    elif epilogue.startswith("gelu"):
        # its slope is at most 1.13; its own 32-bit arithmetic is good to some ten roundings of its argument's size
        off, y = 1.13 * off + 12 * 2.0 ** -24 * y.abs(), gelu(y, epilogue)
    if out_dtype == torch.bfloat16:
        off = off + 2.0 ** -8 * y.abs()
    assert ((out.double() - y).abs() <= off + 1e-30).all()


# one row to several tiles of them, outputs and inputs that end inside a tile and a block of K, one output; K of one piece
@pytest.mark.parametrize("m,n,k", [(1, 1, 16), (1, 4800, 1600), (2, 33, 48), (3, 64, 64), (8, 257, 1024), (16, 128, 6400), (17, 100, 272), (31, 2304, 768), (33, 96, 1040),
                                   (64, 200, 256), (65, 130, 64), (100, 300, 512), (128, 256, 128), (129, 257, 400), (200, 1000, 1600), (257, 513, 144), (700, 64, 2064)])
@pytest.mark.parametrize("dtype,epilogue", [("bfloat16", "store"), ("float32", "store"), ("bfloat16", "gelu_tanh"), ("float32", "gelu_erf"), ("bfloat16", "residual"),
                                            ("bfloat16", "store_f32")])
def test_products(m, n, k, dtype, epilogue):
    check_product(dtype, m, n, k, epilogue)


# every form on its own: tiles of rows and outputs in part, more tiles than SMs, K of one block and of many
@pytest.mark.parametrize("form,m,n,k", [(1, 1, 40, 32), (1, 13, 70, 1616), (1, 16, 40, 6416), (1, 3, 50, 2064), (64, 1, 100, 16), (64, 300, 9000, 144), (128, 40, 129, 256), (128, 500, 6000, 128), (256, 3, 3, 1040), (512, 3, 3, 16), (512, 300, 500, 1040), (512, 129, 70, 48),
                                        (512, 2700, 2304, 640),
                                        (256, 1100, 5000, 272), (256, 2500, 4800, 400)])
@pytest.mark.parametrize("dtype,epilogue", [("bfloat16", "store"), ("float32", "store"), ("bfloat16", "residual")])
def test_products_by_form(form, m, n, k, dtype, epilogue):
    check_product(dtype, m, n, k, epilogue, form=form)


@pytest.mark.parametrize("m", [1, 9, 40, 150])
@pytest.mark.parametrize("dtype,epilogue", [("float32", "gelu_tanh"), ("bfloat16", "gelu_erf"), ("float32", "residual")])
@pytest.mark.parametrize("bias", [None, "bfloat16"])
def test_products_of_rows_that_lie_apart(m, dtype, epilogue, bias):
    check_product(dtype, m, 150, 208, epilogue, bias, extra=16)


@pytest.mark.parametrize("m", [1, 20, 130])
def test_the_largest_sums_are_exact(m):
    k, n = 133136, 70
    a = torch.full((m, k), -127, dtype=torch.int8, device="cuda")
    w = torch.full((n, k), -127, dtype=torch.int8, device="cuda")
    w[1::2] = 127
    out = torch.empty(m, n, device="cuda")
    ops = Ops(torch.float32)
    ops.linear_int8(a, torch.ones(m, device="cuda"), w, torch.ones(n, device="cuda"), None, out)
    want = torch.full((n,), float(k * 127 * 127), device="cuda")
    want[1::2] *= -1
    assert torch.equal(out, want.expand(m, n))


@pytest.mark.parametrize("m", [2, 30, 200])
def test_a_scale_that_is_not_finite_stays_with_its_row_and_output(m):
    a, sa, w, sw, b = product(8, m, 90, 128)
    sa[1], sw[7] = float("nan"), float("nan")
    out = torch.empty(m, 90, device="cuda")
    Ops(torch.float32).linear_int8(a, sa, w, sw, b, out)
    bad = torch.zeros(m, 90, dtype=torch.bool, device="cuda")
    bad[1], bad[:, 7] = True, True
    assert torch.equal(out.isnan(), bad)


# -- the cache ----------------------------------------------------------------------------------------------------------------


class Step:
    """A step's rows and pages dealt out in no order; what nobody has written holds codes and scales that spoil whatever reads them."""

    def __init__(self, new, held_before, kv_heads, hd, seed=0, pool=None):
        lens = [a + b for a, b in zip(new, held_before)]
        n_pages = [-(-n // PAGE) for n in lens]
        self.new, self.lens, self.kv_heads, self.hd = new, lens, kv_heads, hd
        total = sum(n_pages) + 3
        pool = pool or total
        order = (pool - total + torch.randperm(total, generator=torch.Generator().manual_seed(seed))).int()
        table = torch.full((len(new), max(n_pages) + 2), int(order[-1]), dtype=torch.int32)
        at = 0
        for s, n in enumerate(n_pages):
            table[s, :n] = order[at:at + n]
            at += n
        self.table = table.cuda()
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        self.rows, self.n_seqs, self.max_new = starts[-1], len(new), max(new)
        ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
        self.starts, self.kv_lens = ints(starts), ints(lens)
        self.row_seq = ints([s for s, n in enumerate(new) for _ in range(n)])
        self.row_pos = ints([p + i for n, p in zip(new, held_before) for i in range(n)])
        cells = (pool, kv_heads, PAGE)
        self.k, self.v = (torch.empty(*cells, hd, dtype=torch.int8, device="cuda") for _ in range(2))
        self.ks, self.vs = (torch.empty(cells, device="cuda") for _ in range(2))
        for t, x in ((self.k, 127), (self.v, 127), (self.ks, float("nan")), (self.vs, float("nan"))):
            t[pool - total:] = x

    def cells(self, seq):
        """(page, place) of every position of a sequence."""
        pos = torch.arange(self.lens[seq], device="cuda")
        return self.table[seq, pos // PAGE].long(), pos % PAGE

    def fill(self, seed):
        """Every sequence's keys and values in codes; returns them as 64-bit numbers [positions, heads, hd] a sequence."""
        g, got = generator(seed), []
        for s in range(self.n_seqs):
            page, place = self.cells(s)
            pair = []
            for t, sc in ((self.k, self.ks), (self.v, self.vs)):
                codes, scales = held(torch.randn(self.lens[s], self.kv_heads, self.hd, device="cuda", generator=g) * (0.2 + torch.rand(self.lens[s], self.kv_heads, 1, device="cuda", generator=g)))
                t[page, :, place], sc[page, :, place] = codes.to(torch.int8), scales
                pair.append(codes.double() * scales.double().unsqueeze(-1))
            got.append(pair)
        return got

    def pages(self):
        return self.k, self.ks, self.v, self.vs


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("kv_heads,hd", [(1, 16), (3, 32), (12, 64), (2, 48), (8, 128), (1, 80), (2, 256), (5, 144)])
@pytest.mark.parametrize("new,before", [([1], [0]), ([1, 1, 1], [63, 64, 500]), ([3, 130, 1, 64], [62, 0, 7, 64])])
@pytest.mark.parametrize("lead", [0, 24, 1])
def test_keys_and_values_are_written_as_codes_and_read_back(dtype, kv_heads, hd, new, before, lead):
    step, width = Step(new, before, kv_heads, hd), kv_heads * hd
    rows = torch.randn(step.rows, 2 * width + lead, device="cuda", generator=generator(hd)).to(DT[dtype])
    rows[0, lead:lead + hd] = 0                                     # a key of zeros
    k, v = rows[:, lead:lead + width], rows[:, lead + width:]
    untouched = [t.clone() for t in step.pages()]
    ops = Ops(DT[dtype])
    ops.kv_store_int8(k, v, step.row_seq, step.row_pos, step.table, *step.pages())
    page, place = step.table[step.row_seq.long(), step.row_pos.long() // PAGE].long(), step.row_pos.long() % PAGE
    outs = [apart(torch.zeros(step.rows, width, dtype=DT[dtype], device="cuda"), lead) if lead else torch.zeros(step.rows, width, dtype=DT[dtype], device="cuda") for _ in range(2)]
    ops.kv_read_int8(step.row_seq, step.row_pos, step.table, *step.pages(), *outs)
    for src, codes_at, scales_at, out in ((k, step.k, step.ks, outs[0]), (v, step.v, step.vs, outs[1])):
        codes, scales = held(src.float().reshape(step.rows, kv_heads, hd))
        assert torch.equal(codes_at[page, :, place].float(), codes)
        assert torch.equal(scales_at[page, :, place], scales)
        assert torch.equal(out, (codes * scales.unsqueeze(-1)).reshape(step.rows, width).to(DT[dtype]))
    for t, was in zip(step.pages(), untouched):                     # nobody else's places are written
        t[page, :, place] = was[page, :, place]
        assert torch.equal(t, was) or (t.isnan() == was.isnan()).all()


def test_a_key_that_is_not_finite_says_so():
    step = Step([4], [0], 2, 64)
    rows = torch.randn(4, 256, device="cuda", generator=generator(2))
    rows[1, 70], rows[2, 200] = float("inf"), float("nan")          # the second head's key of row 1, the second head's value of row 2
    Ops(torch.float32).kv_store_int8(rows[:, :128], rows[:, 128:], step.row_seq, step.row_pos, step.table, *step.pages())
    page = int(step.table[0, 0])
    assert step.ks[page, :, :4].isnan().nonzero().tolist() == [[1, 1]] and step.vs[page, :, :4].isnan().nonzero().tolist() == [[1, 2]]
    assert (step.k[page, 1, 1] == 0).all() and (step.v[page, 1, 2] == 0).all()


# -- attention ----------------------------------------------------------------------------------------------------------------


def attention_in_64_bits(step, kv, q, n_heads, scale, window, keep_first, places=16):
    """(what each row gets, sum of weight x |value| over the sum of weights, how far the scores can be off in their products' last place)."""
    hd, group = step.hd, n_heads // step.kv_heads
    out = torch.zeros(step.rows, n_heads, hd, dtype=torch.float64, device="cuda")
    size, slack = torch.zeros_like(out), torch.zeros(step.rows, n_heads, 1, dtype=torch.float64, device="cuda")
    at = 0
    for s, (new, length) in enumerate(zip(step.new, step.lens)):
        if not new:
            continue
        i = torch.arange(length - new, length, device="cuda").unsqueeze(1)
        j = torch.arange(length, device="cuda")
        seen = j <= i
        if window:
            seen &= (i - j < window) | (j < keep_first)
        for h in range(n_heads):
            k, v = kv[s][0][:, h // group], kv[s][1][:, h // group]
            rows = q[at:at + new, h * hd:(h + 1) * hd].double()
            scores = ((rows @ k.T) * scale).masked_fill(~seen, -math.inf)
            w = torch.softmax(scores, -1)
            out[at:at + new, h], size[at:at + new, h] = w @ v, w @ v.abs()
            slack[at:at + new, h, 0] = ((rows.abs() @ k.abs().T) * scale).masked_fill(~seen, 0).amax(-1)
        at += new
    return out.view(step.rows, -1), size.view(step.rows, -1), slack.expand(-1, -1, hd).reshape(step.rows, -1)


def check_attention(dtype, new, before, n_heads, kv_heads, hd, window=0, keep_first=0, lead=0, spread=2.0, pool=None, seed=0):
    step = Step(new, before, kv_heads, hd, seed, pool)
    kv = step.fill(seed + 1)
    q = (spread * torch.randn(step.rows, n_heads * hd + lead, device="cuda", generator=generator(seed + 2))).to(DT[dtype])[:, lead:]
    out = torch.full((step.rows, n_heads * hd + lead), float("nan"), dtype=DT[dtype], device="cuda")[:, lead:]
    scale = 1 / math.sqrt(hd)
    Ops(DT[dtype]).attention_int8(q, out, step.starts, step.kv_lens, step.n_seqs, step.max_new, step.table, *step.pages(), n_heads, scale, window=window,
                                  keep_first=keep_first)
    want, size, slack = attention_in_64_bits(step, kv, q, n_heads, scale, window, keep_first)
    # scores: a sum of hd products, each rounding it by 2^-24 of the terms' size at most, and the key's scale; the exponential turns that into a
    # relative error of a weight, twice (in the sum of weights too); sums over the keys; with bfloat16 the weights and the output have 8 bits
    u = U[dtype]
    off = 2 * (hd + 8) * 2.0 ** -24 * slack * size + (64 + 8) * 2.0 ** -23 * size
    if dtype == "bfloat16":
        off = off + u * (size + want.abs())
    got = out.double()
    assert not got.isnan().any()
    assert ((got - want).abs() <= off).all(), float(((got - want).abs() / off).max())
    # and together: roundings of either sign, 0.6 of a unit at most where weights and outputs are rounded (0.41 each)
    rel = float((got - want).norm() / want.norm())
    assert rel <= (0.75 * u if dtype == "bfloat16" else 24 * u), rel


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("n_heads,kv_heads,hd", [(2, 2, 16), (4, 1, 32), (3, 3, 48), (12, 12, 64), (8, 2, 64), (6, 2, 80), (3, 1, 96), (2, 1, 112), (8, 2, 128), (4, 4, 128),
                                                 (5, 1, 144), (16, 1, 64), (20, 1, 128), (2, 2, 192), (4, 2, 256)])
@pytest.mark.parametrize("before", [[0], [62, 63, 64, 65, 0, 300], [700, 650], [1500, 3, 700]])
def test_attention_of_single_tokens(dtype, n_heads, kv_heads, hd, before):
    check_attention(dtype, [1] * len(before), before, n_heads, kv_heads, hd, lead=8)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("n_heads,kv_heads,hd", [(2, 2, 16), (4, 1, 32), (3, 3, 48), (4, 4, 64), (8, 2, 64), (6, 2, 80), (3, 1, 96), (2, 1, 112), (8, 2, 128), (4, 4, 128),
                                                 (5, 1, 144), (2, 2, 192), (4, 2, 256)])
@pytest.mark.parametrize("new,before", [([2], [0]), ([63, 64, 65], [0, 0, 0]), ([1, 130, 17, 5], [70, 0, 200, 59]), ([300], [129])])
def test_attention_of_prompts_and_chunks(dtype, n_heads, kv_heads, hd, new, before):
    check_attention(dtype, new, before, n_heads, kv_heads, hd, lead=8)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("hd", [64, 128, 80])
@pytest.mark.parametrize("window,keep_first", [(1, 0), (1, 1), (20, 4), (64, 70), (100, 0), (128, 64), (1000, 3), (5, 2000)])
@pytest.mark.parametrize("new,before", [([1, 1, 1], [200, 63, 1000]), ([150, 3], [0, 333])])
def test_attention_with_a_window_and_kept_positions(dtype, hd, window, keep_first, new, before):
    check_attention(dtype, new, before, 4, 2, hd, window, keep_first)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("hd", [64, 128])
def test_rows_that_lie_apart_and_off_the_boundaries(dtype, hd):
    check_attention(dtype, [1, 1], [100, 5], 4, 2, hd, lead=3)
    check_attention(dtype, [70, 10], [100, 5], 4, 2, hd, lead=3)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_a_sequence_without_new_rows(dtype):
    check_attention(dtype, [0, 70, 0, 2, 0], [50, 10, 3, 64, 1], 4, 2, 64)
    check_attention(dtype, [0, 1, 0, 1], [50, 10, 3, 64], 4, 2, 64)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("new", [1, 90])
def test_long_contexts(dtype, new):
    check_attention(dtype, [new], [9000], 4, 2, 128)
    check_attention(dtype, [new, new], [6000, 40], 2, 2, 64, spread=6.0)


@pytest.mark.parametrize("seqs,longest,n_heads,kv_heads,hd,window", [(40, 200, 8, 4, 64, 0), (33, 300, 8, 8, 128, 0), (40, 200, 4, 4, 64, 100), (260, 4, 2, 1, 16, 0), (300, 1, 2, 2, 64, 0)])
def test_more_blocks_than_multiprocessors(seqs, longest, n_heads, kv_heads, hd, window):
    """Blocks come in the order of the pages they see, which each finds for itself (up to 256 sequences); some sequences have no new rows."""
    g = torch.Generator().manual_seed(seqs)
    new = [int(x) for x in torch.randint(0, longest + 1, (seqs,), generator=g)]
    new[3], new[5] = longest, 0
    before = [int(x) + (n == 0) for x, n in zip(torch.randint(0, 700, (seqs,), generator=g), new)]
    check_attention("bfloat16", new, before, n_heads, kv_heads, hd, window)


@pytest.mark.parametrize("new", [[1, 1], [80, 1]])
def test_pages_beyond_two_thousand_million_bytes(new):
    check_attention("bfloat16", new, [200, 10], 8, 8, 128, pool=(1 << 31) // (8 * PAGE * 128) + 40)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("hd", [64, 128, 80])
@pytest.mark.parametrize("which", ["key", "value"])
@pytest.mark.parametrize("new,before", [([100], [90]), ([1, 1], [150, 100])])
def test_a_row_that_is_not_finite_reaches_those_who_see_it_alone(dtype, hd, which, new, before):
    step = Step(new, before, 2, hd)
    step.fill(3)
    at = 120                                                        # of the first sequence, in the first head
    page, place = step.cells(0)
    (step.ks if which == "key" else step.vs)[page[at], 0, place[at]] = float("nan")
    q = torch.randn(step.rows, 4 * hd, device="cuda", generator=generator(4)).to(DT[dtype])
    out = torch.zeros(step.rows, 4, hd, dtype=DT[dtype], device="cuda")
    Ops(DT[dtype]).attention_int8(q, out.view(step.rows, -1), step.starts, step.kv_lens, step.n_seqs, step.max_new, step.table, *step.pages(), 4, 0.1)
    bad = torch.zeros(step.rows, 4, dtype=torch.bool, device="cuda")
    bad[:, :2] = ((step.row_seq == 0) & (step.row_pos >= at)).unsqueeze(1)
    assert torch.equal(out.isnan().all(-1), bad) and torch.equal(out.isnan().any(-1), bad)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("new,before", [([60], [40]), ([1], [99])])
def test_scales_of_all_sizes(dtype, new, before):
    """Keys and values of zeros, and values whose scales are nine orders of magnitude apart: each row's error follows what it sums."""
    step = Step(new, before, 1, 64)
    kv = step.fill(5)
    page, place = step.cells(0)
    factor = torch.ones(100, dtype=torch.float64, device="cuda")
    factor[::7], factor[3::9], factor[2] = 0, 2.0 ** -30, 2.0 ** 12
    step.vs[page, 0, place] *= factor.float()
    kv[0][1] *= factor.view(-1, 1, 1)
    step.ks[page[5], 0, place[5]] = 0
    kv[0][0][5] = 0
    q = torch.randn(step.rows, 128, device="cuda", generator=generator(6)).to(DT[dtype])
    out = torch.zeros(step.rows, 128, dtype=DT[dtype], device="cuda")
    Ops(DT[dtype]).attention_int8(q, out, step.starts, step.kv_lens, 1, step.max_new, step.table, *step.pages(), 2, 0.125)
    want, size, slack = attention_in_64_bits(step, kv, q, 2, 0.125, 0, 0)
    off = 2 * 72 * 2.0 ** -24 * slack * size + 72 * 2.0 ** -23 * size + (U[dtype] * (size + want.abs()) if dtype == "bfloat16" else 0)
    assert ((out.double() - want).abs() <= off).all()


def test_what_a_row_gets_does_not_depend_on_the_others():
    """The same sequence alone and beside others, single tokens and a chunk."""
    for new in (1, 70):
        got = []
        for others in ([], [(1, 500)], [(1, 3)] * 30):
            step = Step([new] + [n for n, _ in others], [333] + [b for _, b in others], 2, 64)
            g = torch.Generator().manual_seed(1)
            page, place = step.cells(0)
            for t, sc in ((step.k, step.ks), (step.v, step.vs)):
                t[page, :, place] = torch.randint(-127, 128, (333 + new, 2, 64), generator=g, dtype=torch.int8).cuda()
                sc[page, :, place] = torch.rand(333 + new, 2, generator=g).cuda() * 0.01
            q = torch.randn(step.rows, 256, generator=torch.Generator().manual_seed(2)).cuda().bfloat16()
            q[:new] = torch.randn(new, 256, generator=g).cuda().bfloat16()
            for s in range(1, step.n_seqs):
                page, place = step.cells(s)
                step.ks[page, :, place] = step.vs[page, :, place] = 0.01
            out = torch.zeros(step.rows, 256, dtype=torch.bfloat16, device="cuda")
            Ops(torch.bfloat16).attention_int8(q, out, step.starts, step.kv_lens, step.n_seqs, new, step.table, *step.pages(), 4, 0.125)
            got.append(out[:new].double())
        for other in got[1:]:
            assert (got[0] - other).norm() <= 2.0 ** -8 * got[0].norm()       # (how the keys are dealt out may differ with the batch)


# -- refusals and streams -------------------------------------------------------------------------------------------------------


def test_refusals():
    ops = Ops(torch.bfloat16)
    i8 = lambda *s: torch.zeros(*s, dtype=torch.int8, device="cuda")
    f = lambda *s: torch.zeros(*s, device="cuda")
    h = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device="cuda")
    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")

    def refused(what, *words):
        with pytest.raises(KernelError) as e:
            what()
        assert all(w in str(e.value) for w in words), str(e.value)

    refused(lambda: ops.int8_rows(f(2, 8).cpu(), i8(2, 8), f(2)), "CUDA tensors only")
    refused(lambda: ops.int8_rows(f(2, 8), h(2, 8), f(2)), "codes must be int8")
    refused(lambda: ops.int8_rows(f(2, 8), i8(2, 8), f(3)), "one per row")
    refused(lambda: ops.int8_rows(f(2, 8).half(), i8(2, 8), f(2)), "float32 or bfloat16")
    refused(lambda: ops.int8_rows(f(1, 32772), i8(1, 32772), f(1)), "at most 32768")
    refused(lambda: ops.int8_rows(f(0, 8), i8(0, 8), f(0)), "needs rows")
    refused(lambda: ops.rmsnorm_int8(h(2, 8), None, 1e-5, i8(2, 8), f(2)), "float32 residual stream")
    refused(lambda: ops.rmsnorm_int8(f(2, 8), f(7), 1e-5, i8(2, 8), f(2)), "row's width")
    refused(lambda: ops.layernorm_int8(f(2, 8), f(8), h(8), 1e-5, i8(2, 8), f(2)), "one dtype")
    refused(lambda: ops.rmsnorm_int8(f(2, 8), None, 1e-5, i8(1, 8), f(1), rows=i(1), delta=f(2, 8)), "goes without a sum")
    refused(lambda: ops.rmsnorm_int8(f(2, 8), None, 1e-5, i8(2, 8), f(2), delta=f(2, 7)), "stream's shape")
    refused(lambda: ops.int8_read(i8(2, 8), f(2), torch.zeros(2, 8, dtype=torch.float16, device="cuda")), "float32 or bfloat16")
    refused(lambda: ops.linear_int8(i8(2, 24), f(2), i8(4, 24), f(4), None, h(2, 4)), "multiple of 16")
    refused(lambda: ops.linear_int8(i8(2, 32), f(2), i8(4, 16), f(4), None, h(2, 4)), "does not take inputs")
    refused(lambda: ops.linear_int8(i8(2, 32), f(2), i8(4, 32), f(3), None, h(2, 4)), "one per output")
    refused(lambda: ops.linear_int8(i8(2, 32), f(2), i8(4, 32), f(4), None, f(2, 4)), "output must be")
    refused(lambda: ops.linear_int8(i8(2, 32), f(2), i8(4, 32), f(4), f(5), h(2, 4)), "bias")
    refused(lambda: ops.linear_int8(i8(2, 33)[:, 1:], f(2), i8(4, 32), f(4), None, h(2, 4)), "16-byte boundaries")
    cache = lambda hd=64, page=64: (i8(3, 2, page, hd), f(3, 2, page), i8(3, 2, page, hd), f(3, 2, page))
    refused(lambda: ops.kv_store_int8(h(1, 128), f(1, 128), i(1), i(1), i(1, 2), *cache()), "views")
    refused(lambda: ops.kv_store_int8(h(1, 144), h(1, 144), i(1), i(1), i(1, 2), *cache(72)), "multiples of 16")
    refused(lambda: ops.kv_store_int8(h(1, 128), h(1, 128), i(1).long(), i(1), i(1, 2), *cache()), "int32")
    refused(lambda: ops.kv_read_int8(i(1), i(1), i(1, 2), *cache(), h(1, 128), h(1, 64)), "must be")
    attend = lambda q, o, c, heads=4, **kw: ops.attention_int8(q, o, i(2), i(1), 1, 1, i(1, 2), *c, heads, 0.125, **kw)
    refused(lambda: attend(h(1, 256), h(1, 255), cache()), "heads x head size")
    refused(lambda: attend(f(1, 256), f(1, 256), cache()), "must be torch.bfloat16")
    refused(lambda: attend(h(1, 192), h(1, 192), cache(), 3), "do not divide")
    refused(lambda: attend(h(1, 4 * 272), h(1, 4 * 272), cache(272)), "up to 256")
    refused(lambda: attend(h(1, 256), h(1, 256), cache(page=32)), "64 positions")
    refused(lambda: attend(h(1, 256), h(1, 256), cache(), window=-1), "negative")
    refused(lambda: attend(h(1, 256), h(1, 256), (h(3, 2, 64, 64),) + cache()[1:]), "int8")


def test_another_stream():
    ops, stream = Ops(torch.bfloat16), torch.cuda.Stream()
    a, sa, w, sw, b = product(3, 200, 300, 256)
    want = torch.empty(200, 300, device="cuda")
    ops.linear_int8(a, sa, w, sw, b, want, "store_f32")
    x = torch.randn(200, 256, device="cuda")
    torch.cuda.synchronize()
    got, codes, scales = torch.empty_like(want), torch.empty(200, 256, dtype=torch.int8, device="cuda"), torch.empty(200, device="cuda")
    with torch.cuda.stream(stream):
        torch.cuda._sleep(2_000_000)
        x.mul_(2)
        ops.int8_rows(x, codes, scales)
        ops.linear_int8(a, sa, w, sw, b, got, "store_f32")
    stream.synchronize()
    assert torch.equal(got, want) and torch.equal(scales, held(x)[1])
