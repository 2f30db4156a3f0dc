"""Cases that stand for work in 8-bit integers: rows normed and held as codes with one scale each, products of such rows with
weights held the same way, keys and values held so in the paged cache as they are written, and attention that reads them.

A row x is held as codes c (integers of -127 .. 127) and a 32-bit scale s = max|x| / 127: x ~ c s, c = x / s rounded to the nearest
integer, halves to the even one; a row of zeros has the scale 0.  A row of activations has one scale, a row of weights (one output)
has one, a position's key or value has one for each key/value head.

Sizes are those of the benchmark's models (widths of 768 to 1600 with heads of 64, GPT-2 XL's products) and of generic designs with
grouped heads of 128.  `lengths` and `cached` are texts of numbers, one per sequence: the rows it brings, and the positions it held before.
"""
import functools
import math

import torch

own = False

PAGE = 64
DT = {"bfloat16": torch.bfloat16, "float32": torch.float32}


def listed():
    long = " ".join(str(1000 + i * 2741 % 7193) for i in range(64))
    return [
        # what a sublayer of a decoding step left is added to the stream, and the stream normed for the next product: 8 sequences
        dict(name="norm_step", kind="norm", norm="rms", rows=8, width=1024, delta=True, weight="float32"),
        # the same of a batch of long prompts
        dict(name="norm_prompts", kind="norm", norm="rms", rows=16384, width=4096, delta=True, weight="bfloat16"),
        # q, k and v of eight decoding sequences at GPT-2 XL's sizes: a stream of weights
        dict(name="product_step", kind="product", rows=8, n_in=1600, n_out=4800, epilogue="store", bias=True, dtype="bfloat16"),
        # the way up of a ragged batch of a few short prompts at GPT-2 medium's sizes, in the 32-bit engine
        dict(name="product_ragged_f32", kind="product", rows=333, n_in=1024, n_out=4096, epilogue="gelu_erf", bias=True, dtype="float32"),
        # the way up of two whole contexts at GPT-2 XL's sizes
        dict(name="product_prompt", kind="product", rows=2048, n_in=1600, n_out=6400, epilogue="gelu_tanh", bias=True, dtype="bfloat16"),
        # a wide product of long prompts, with 32-bit results
        dict(name="product_large", kind="product", rows=8192, n_in=4096, n_out=8192, epilogue="store_f32", bias=False, dtype="bfloat16"),
        # keys and values of a decoding step: 8 sequences of GPT-2 small, written to the cache and read back
        dict(name="cache_step", kind="cache", lengths="1 1 1 1 1 1 1 1", cached="519 511 530 522 498 540 515 527", kv_heads=12, head_dim=64,
             dtype="bfloat16"),
        # keys and values of long prompts, some of them behind others, as when a sequence is taken out of the cache for a while
        dict(name="cache_prompts", kind="cache", lengths="8000 4097 6001 8191", cached="0 100 1000 1", kv_heads=8, head_dim=128, dtype="bfloat16"),
        # a decoding step of GPT-2 small: 8 sequences after about 520 positions
        dict(name="attend_step", kind="attend", lengths="1 1 1 1 1 1 1 1", cached="519 511 530 522 498 540 515 527", heads=12, kv_heads=12,
             head_dim=64, window=0, keep_first=0, dtype="bfloat16"),
        # a decoding step of 64 long sequences with grouped heads: a stream of the cache
        dict(name="attend_long_step", kind="attend", lengths=" ".join(["1"] * 64), cached=long, heads=32, kv_heads=8, head_dim=128, window=0,
             keep_first=0, dtype="bfloat16"),
        # two whole contexts at GPT-2 medium's head sizes
        dict(name="attend_prompt", kind="attend", lengths="1024 1024", cached="0 0", heads=16, kv_heads=16, head_dim=64, window=0, keep_first=0,
             dtype="bfloat16"),
        # chunks of new tokens behind long ragged contexts, grouped heads
        dict(name="attend_chunks", kind="attend", lengths="512 512 509 512", cached="7680 4096 6002 1024", heads=32, kv_heads=8, head_dim=128,
             window=0, keep_first=0, dtype="bfloat16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi, multiple=1):
    n = max(multiple, _log(rng, lo, hi) // multiple * multiple)
    return n + multiple if n == 3072 else n


def draw(rng):
    kind = rng.choice(["norm", "product", "product", "cache", "attend", "attend"])
    if kind == "norm":
        width = _size(rng, 48, 6400, rng.choice([1, 8, 16, 64]))
        return dict(kind=kind, norm=rng.choice(["rms", "layer"]), rows=min(_log(rng, 1, 16384), (16384 * 4096) // width), width=width,
                    delta=rng.random() < 0.7, weight=rng.choice(["float32", "bfloat16"]))
    if kind == "product":
        n_in, n_out = _size(rng, 64, 6400, 16), _size(rng, 64, 8192, rng.choice([1, 8, 16, 64]))
        rows = min(_log(rng, 1, 8192), (8192 * 4096 * 8192) // (n_in * n_out))
        return dict(kind=kind, rows=rows, n_in=n_in, n_out=n_out, epilogue=rng.choice(["store", "gelu_tanh", "gelu_erf", "store_f32"]),
                    bias=rng.random() < 0.7, dtype=rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"]))
    hd = rng.choice([16, 32, 64, 64, 64, 80, 96, 128, 128, 128, 256])
    dtype = rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"])
    if kind == "cache":
        seqs, kv = rng.randint(1, 8), rng.randint(1, 16)
        most = max(1, min(8192, 8 * 128 * 26289 // (kv * hd * seqs)))
        new = [_log(rng, 1, most) for _ in range(seqs)] if rng.random() < 0.7 else [1] * seqs
        return dict(kind=kind, lengths=" ".join(map(str, new)), cached=" ".join(str(rng.randint(0, 2000)) for _ in new), kv_heads=kv, head_dim=hd,
                    dtype=dtype)
    kv, group = rng.choice([1, 2, 4, 8, 12]), rng.choice([1, 1, 2, 3, 4, 8])
    window = rng.choice([0, 0, 0, _log(rng, 16, 2048)])
    keep = rng.choice([0, 4, 70]) if window else 0
    if rng.random() < 0.5:                      # single tokens
        seqs = _log(rng, 1, 64)
        new, held = [1] * seqs, [_log(rng, 1, min(8192, (64 * 4600 * 8 * 128) // (seqs * kv * hd))) for _ in range(seqs)]
    else:                                       # prompts, and chunks of them behind what is there
        seqs = rng.randint(1, 6)
        new = [_log(rng, 1, 1024) for _ in range(seqs)]
        held = [rng.choice([0, 0, rng.randint(1, 2000)]) for _ in range(seqs)]
    return dict(kind=kind, lengths=" ".join(map(str, new)), cached=" ".join(map(str, held)), heads=kv * group, kv_heads=kv, head_dim=hd,
                window=window, keep_first=keep, dtype=dtype)


# -- inputs ---------------------------------------------------------------------------------------------------------------


def _codes(x):
    """Rows (the last axis) as codes and scales, in the input's precision."""
    top = x.abs().amax(-1)
    scales = top * (1 / 127)
    codes = torch.round(x / torch.where(scales > 0, scales, 1).unsqueeze(-1)).clamp(-127, 127)
    return codes, scales


def _held(gen, dev, *shape):
    """Rows of ordinary numbers, held in 8 bits."""
    codes, scales = _codes(torch.randn(*shape, device=dev, generator=gen))
    return codes.to(torch.int8), scales


def _step(case, gen, dev):
    """A step's rows and where they stand: pages dealt out in no order, with some to spare."""
    new, held = ([int(x) for x in case[key].split()] for key in ("lengths", "cached"))
    lens = [a + b for a, b in zip(new, held)]
    n_pages = [-(-n // PAGE) for n in lens]
    spare, width = 5, max(n_pages)
    order = torch.randperm(sum(n_pages) + spare, device=dev, generator=gen).to(torch.int32)
    table = torch.zeros(len(new), width, dtype=torch.int32, device=dev)
    at = 0
    for s, n in enumerate(n_pages):
        table[s, :n] = order[at:at + n]
        at += n
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    ints = functools.partial(torch.tensor, dtype=torch.int32, device=dev)
    new_t, held_t = ints(new).long(), ints(held).long()
    row_seq = torch.repeat_interleave(torch.arange(len(new), device=dev), new_t)
    row_pos = torch.arange(starts[-1], device=dev) - ints(starts).long()[row_seq] + held_t[row_seq]
    return {"rows": starts[-1], "n_seqs": len(new), "max_new": max(new), "pool": sum(n_pages) + spare, "table": table, "seq_starts": ints(starts),
            "kv_lens": ints(lens), "row_seq": row_seq.to(torch.int32), "row_pos": row_pos.to(torch.int32)}


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(dev).manual_seed(int(seed))

    def randn(*shape):
        return torch.randn(*shape, device=dev, generator=gen)

    state = {"case": case}
    if case["kind"] == "norm":
        rows, width = case["rows"], case["width"]
        # a stream has a few channels that are much larger than the others
        loud = 1 + 8 * (torch.rand(width, device=dev, generator=gen) < 0.01)
        state |= {"x": randn(rows, width) * loud + 0.1, "delta": (0.3 * randn(rows, width)).bfloat16() if case["delta"] else None,
                  "weight": (1 + 0.05 * randn(width)).to(DT[case["weight"]]),
                  "bias": (0.02 * randn(width)).to(DT[case["weight"]]) if case["norm"] == "layer" else None,
                  "x_out": torch.empty(rows, width, device=dev), "codes": torch.empty(rows, width, dtype=torch.int8, device=dev),
                  "scales": torch.empty(rows, device=dev), "values": torch.empty(rows, width, dtype=torch.bfloat16, device=dev)}
    elif case["kind"] == "product":
        a, a_scales = _held(gen, dev, case["rows"], case["n_in"])
        w, w_scales = _held(gen, dev, case["n_out"], case["n_in"])
        out = torch.float32 if case["epilogue"] == "store_f32" else DT[case["dtype"]]
        state |= {"a": a, "a_scales": a_scales, "w": w, "w_scales": w_scales * (2 / math.sqrt(case["n_in"])),
                  "bias": 0.1 * randn(case["n_out"]) if case["bias"] else None,
                  "out": torch.empty(case["rows"], case["n_out"], dtype=out, device=dev)}
    else:
        state |= _step(case, gen, dev)
        kv, hd, dtype = case["kv_heads"], case["head_dim"], DT[case["dtype"]]
        pages = (state["pool"], kv, PAGE)
        if case["kind"] == "cache":
            # keys and values are columns of the product that gave them and the queries; keys have loud channels of their own
            rows = randn(state["rows"], 3 * kv * hd)
            rows[:, kv * hd:2 * kv * hd] *= 1 + 4 * (torch.rand(kv * hd, device=dev, generator=gen) < 0.05)
            rows = rows.to(dtype)
            state |= {"k": rows[:, kv * hd:2 * kv * hd], "v": rows[:, 2 * kv * hd:],
                      "k_pages": torch.zeros(*pages, hd, dtype=torch.int8, device=dev), "k_scales": torch.zeros(pages, device=dev),
                      "v_pages": torch.zeros(*pages, hd, dtype=torch.int8, device=dev), "v_scales": torch.zeros(pages, device=dev),
                      "k_out": torch.empty(state["rows"], kv * hd, dtype=dtype, device=dev),
                      "v_out": torch.empty(state["rows"], kv * hd, dtype=dtype, device=dev)}
        else:
            state["k_pages"], state["k_scales"] = _held(gen, dev, *pages, hd)
            state["v_pages"], state["v_scales"] = _held(gen, dev, *pages, hd)
            # queries whose scores spread by about 2: some keys count, most hardly
            state |= {"q": (2 * randn(state["rows"], case["heads"] * hd)).to(dtype), "scale": 1 / math.sqrt(hd),
                      "out": torch.empty(state["rows"], case["heads"] * hd, dtype=dtype, device=dev)}
    return state


# -- one pass -------------------------------------------------------------------------------------------------------------


@functools.lru_cache(maxsize=None)
def _ops(dtype):
    from kvad_b200.ops import Ops
    return Ops(DT[dtype])


def run(state):
    c = state["case"]
    return {"norm": _norm, "product": _product, "cache": _cache, "attend": _attend}[c["kind"]](state, c)


def _norm(s, c):
    eps = 1e-5
    if own:
        ops = _ops("bfloat16")
        if c["norm"] == "rms":
            ops.rmsnorm_int8(s["x"], s["weight"], eps, s["codes"], s["scales"], delta=s["delta"], x_out=s["x_out"])
        else:
            ops.layernorm_int8(s["x"], s["weight"], s["bias"], eps, s["codes"], s["scales"], delta=s["delta"], x_out=s["x_out"])
        ops.int8_read(s["codes"], s["scales"], s["values"])
        return {"x": s["x_out"], "scales": s["scales"], "values": s["values"]}
    x = s["x"] if s["delta"] is None else s["x"] + s["delta"].float()
    y = x - x.mean(-1, keepdim=True) if c["norm"] == "layer" else x
    y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + eps) * s["weight"].float()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    codes, scales = _codes(y)
    return {"x": x.clone() if s["delta"] is None else x, "scales": scales, "values": (codes * scales.unsqueeze(-1)).bfloat16()}


def _product(s, c):
    if own:
        _ops(c["dtype"]).linear_int8(s["a"], s["a_scales"], s["w"], s["w_scales"], s["bias"], s["out"], c["epilogue"])
        return s["out"]
    y = (s["a"].float() @ s["w"].float().T) * s["a_scales"].unsqueeze(1) * s["w_scales"]
    if s["bias"] is not None:
        y = y + s["bias"]
    if c["epilogue"] == "gelu_tanh":
        y = 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)))
    elif c["epilogue"] == "gelu_erf":
        y = 0.5 * y * (1 + torch.erf(y / math.sqrt(2)))
    return y.to(s["out"].dtype)


def _cache(s, c):
    if own:
        ops = _ops(c["dtype"])
        ops.kv_store_int8(s["k"], s["v"], s["row_seq"], s["row_pos"], s["table"], s["k_pages"], s["k_scales"], s["v_pages"], s["v_scales"])
        ops.kv_read_int8(s["row_seq"], s["row_pos"], s["table"], s["k_pages"], s["k_scales"], s["v_pages"], s["v_scales"], s["k_out"], s["v_out"])
        return {"k": s["k_out"], "v": s["v_out"], "k_scales": s["k_scales"], "v_scales": s["v_scales"]}
    kv, hd = c["kv_heads"], c["head_dim"]
    pos = s["row_pos"].long()
    page, slot = s["table"][s["row_seq"].long(), pos // PAGE].long(), pos % PAGE
    got = {}
    for name in ("k", "v"):
        codes, scales = _codes(s[name].float().view(-1, kv, hd))
        s[name + "_pages"][page, :, slot] = codes.to(torch.int8)
        s[name + "_scales"][page, :, slot] = scales
        values = s[name + "_pages"][page, :, slot].float() * s[name + "_scales"][page, :, slot].unsqueeze(-1)
        got |= {name: values.reshape(-1, kv * hd).to(s[name].dtype), name + "_scales": s[name + "_scales"]}
    return got


def _attend(s, c):
    if own:
        _ops(c["dtype"]).attention_int8(s["q"], s["out"], s["seq_starts"], s["kv_lens"], s["n_seqs"], s["max_new"], s["table"], s["k_pages"], s["k_scales"],
                                        s["v_pages"], s["v_scales"], c["heads"], s["scale"], window=c["window"], keep_first=c["keep_first"])
        return s["out"]
    heads, kv, hd, n, new = c["heads"], c["kv_heads"], c["head_dim"], s["n_seqs"], s["max_new"]
    table = s["table"].long()
    keys, values = ((s[x + "_pages"][table].float() * s[x + "_scales"][table].unsqueeze(-1)).transpose(1, 2).reshape(n, kv, 1, -1, hd)
                    for x in ("k", "v"))
    # every sequence's rows at places of their own, the longest one's number of them
    starts, lens = s["seq_starts"].long(), s["kv_lens"].long()
    first = lens - (starts[1:] - starts[:-1])
    row_seq = s["row_seq"].long()
    row_at = torch.arange(s["rows"], device=table.device) - starts[row_seq]
    q = torch.zeros(n, new, heads * hd, device=table.device)
    q[row_seq, row_at] = s["q"].float()
    q = q.view(n, new, kv, heads // kv, hd).permute(0, 2, 3, 1, 4)
    scores = (q @ keys.transpose(-1, -2)) * s["scale"]
    i = (first.unsqueeze(1) + torch.arange(new, device=table.device)).unsqueeze(2)
    j = torch.arange(keys.shape[3], device=table.device)
    seen = j <= i
    if c["window"]:
        seen &= (i - j < c["window"]) | (j < c["keep_first"])
    scores = scores.masked_fill(~seen.view(n, 1, 1, new, -1), -math.inf)
    weights = torch.exp(scores - scores.amax(-1, keepdim=True))
    out = (weights @ values) / weights.sum(-1, keepdim=True)
    return out.permute(0, 3, 1, 2, 4).reshape(n, new, heads * hd)[row_seq, row_at].to(s["out"].dtype)


# -- what a pass cannot do without, and what it gives in 64 bits -------------------------------------------------------------


def _reach(case):
    """For each sequence: (its new rows, its length, the positions that any of its rows sees, the pairs of row and position)."""
    w, keep = case["window"], case["keep_first"]
    got = []
    for n, p in zip(map(int, case["lengths"].split()), map(int, case["cached"].split())):
        if not w:
            got.append((n, n + p, n + p, n * p + n * (n + 1) // 2))
            continue
        lo = max(0, p - w + 1)                          # the first row's window begins there
        pairs = sum(min(i + 1, w) + min(keep, max(0, i + 1 - w)) for i in range(p, p + n))
        got.append((n, n + p, n + p - lo + min(keep, lo), pairs))
    return got


def work(case):
    kind = case["kind"]
    if kind == "norm":
        rows, width = case["rows"], case["width"]
        # the stream in and out, what is added, the codes, the values they stand for, the scales
        return {"bytes": rows * (width * (4 + 4 + (2 if case["delta"] else 0) + 1 + 2) + 4) + 4 * width, "flops": 10 * rows * width}
    if kind == "product":
        m, k, n = case["rows"], case["n_in"], case["n_out"]
        size = 4 if case["epilogue"] == "store_f32" or case["dtype"] == "float32" else 2
        return {"bytes": m * k + n * k + 4 * (m + 2 * n) + size * m * n, "flops": 2 * m * n * k}
    size, hd = DT[case["dtype"]].itemsize, case["head_dim"]
    if kind == "cache":
        rows = sum(map(int, case["lengths"].split())) * case["kv_heads"] * 2
        return {"bytes": rows * (hd * (2 * size + 1) + 4), "flops": 6 * rows * hd}
    reach = _reach(case)
    rows, seen, pairs = (sum(r[k] for r in reach) for k in (0, 2, 3))
    return {"bytes": 2 * rows * case["heads"] * hd * size + 2 * seen * case["kv_heads"] * (hd + 4), "flops": 4 * pairs * case["heads"] * hd}


def exact(case, seed):
    s = prepare(case, seed)

    def held64(x):
        scale = x.abs().amax(-1, keepdim=True) / 127
        return torch.round(x / scale.clamp_min(1e-300)) * scale, scale.squeeze(-1)

    kind = case["kind"]
    if kind == "norm":
        x = s["x"].double()
        if s["delta"] is not None:
            x = x + s["delta"].double()
        if case["norm"] == "layer":
            mean = x.sum(-1, keepdim=True) / case["width"]
            var = ((x - mean) ** 2).sum(-1, keepdim=True) / case["width"]
            y = (x - mean) / torch.sqrt(var + 1e-5) * s["weight"].double() + s["bias"].double()
        else:
            y = x / torch.sqrt((x ** 2).sum(-1, keepdim=True) / case["width"] + 1e-5) * s["weight"].double()
        values, scales = held64(y)
        return {"x": x, "scales": scales, "values": values}
    if kind == "product":
        got = []
        for lo in range(0, case["rows"], 1024):
            y = (s["a"][lo:lo + 1024].double() * s["a_scales"][lo:lo + 1024].double()[:, None]) @ (s["w"].double() * s["w_scales"].double()[:, None]).T
            if s["bias"] is not None:
                y = y + s["bias"].double()
            if case["epilogue"] == "gelu_tanh":
                y = y / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))
            elif case["epilogue"] == "gelu_erf":
                y = y * 0.5 * torch.erfc(-y / math.sqrt(2))
            got.append(y)
        return torch.cat(got)
    kv, hd = case["kv_heads"], case["head_dim"]
    if kind == "cache":
        got = {}
        for name in ("k", "v"):
            values, scales = held64(s[name].double().view(-1, kv, hd))
            pages = torch.zeros_like(s[name + "_scales"], dtype=torch.float64)
            for r0 in range(0, s["rows"], 4096):
                pos = s["row_pos"][r0:r0 + 4096].long()
                pages[s["table"][s["row_seq"][r0:r0 + 4096].long(), pos // PAGE].long(), :, pos % PAGE] = scales[r0:r0 + 4096]
            got |= {name: values.reshape(-1, kv * hd), name + "_scales": pages}
        return got
    heads, group = case["heads"], case["heads"] // kv
    out = torch.empty(s["rows"], heads, hd, dtype=torch.float64, device=s["q"].device)
    at = 0
    for n, (new, length, _, _) in enumerate(_reach(case)):
        pages = s["table"][n, :-(-length // PAGE)].long()
        i = torch.arange(length - new, length, device=out.device)[:, None]
        j = torch.arange(length, device=out.device)[None]
        seen = (j <= i) & ((i - j < case["window"]) | (j < case["keep_first"])) if case["window"] else j <= i
        for h in range(kv):
            k, v = (s[x + "_pages"][pages, h].double().reshape(-1, hd)[:length] * s[x + "_scales"][pages, h].double().reshape(-1, 1)[:length]
                    for x in ("k", "v"))
            for g in range(h * group, (h + 1) * group):
                scores = (s["q"][at:at + new, g * hd:(g + 1) * hd].double() @ k.T) * s["scale"]
                out[at:at + new, g] = torch.softmax(scores.masked_fill(~seen, -math.inf), -1) @ v
        at += new
    return out.reshape(s["rows"], heads * hd)
