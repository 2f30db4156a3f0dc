"""A GPT-2 whose products and cache are in 8 bits, through the engine, against the same definition in 64 bits."""
import numpy as np
import pytest
import torch

from kvad_b200 import Engine, StepEntry
from tests.conftest import SEEDS, TINY, random_tokens, rel_err
from tests.plain.gpt2_plain import PlainGpt2

pytestmark = pytest.mark.gpu


def held(x):
    """What rows (the last axis) stand for once they are codes and scales."""
    s = np.abs(x).max(axis=-1, keepdims=True) / 127
    return np.rint(x / np.where(s > 0, s, 1)) * s


class Plain8(PlainGpt2):
    @staticmethod
    def linear(x, w_in_out, b):
        return held(x) @ held(w_in_out.T).T + b

    def attention(self, q, k, v, layer, window=None):
        heads = lambda t: held(t.reshape(len(t), self.Hkv, self.hd)).reshape(len(t), -1)
        return super().attention(q, heads(k), heads(v), layer, window)


# How far two runs of one sequence may be apart that cut the work in different ways.  A quotient that lies within its rounding of a half becomes the other code:
# one entry of a row then differs by its scale, max|x| / 127, some 3 / 127 of the row's size, and a product of K of them by 3 / (127 sqrt(K)) of its own: 3e-3 at
# K = 64, and two layers of them.  Where the same kernels run the same rows none does; single rows and many take different ones, whose attention rounds differently, and a
# bfloat16 engine rounds that to 8 bits, a third of a code, before it is quantised.
TOL = {"float32": 6e-3, "bfloat16": 3e-2}


@pytest.fixture(scope="module")
def engines8(model_dirs):
    cache = {}

    def get(name, dtype):
        if (name, dtype) not in cache:
            cache[name, dtype] = Engine.from_pretrained(model_dirs[name], dtype, max_tokens=4096, int8=True)
        return cache[name, dtype]
    return get


def run(engine, pieces):
    """Logits at every place of one sequence fed piece by piece."""
    slot, got = engine.open(), []
    for p in pieces:
        got.append(engine.step([StepEntry(slot, p, range(len(p)))]).cpu().numpy().copy())
    engine.close(slot)
    return np.concatenate(got)


@pytest.mark.parametrize("name", ["A", "B", "D", "A32"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_logits_are_those_of_the_8_bit_definition(engines8, model_dirs, name, dtype):
    """Where a quotient is near a half the engine and 64 bits may take different codes, and what follows in that row is then another draw of the roundings: as far from
    the definition as the definition is from numbers without codes, and twice that at most, since both draws have an error of that size."""
    rounded = "bfloat16" if dtype == "bfloat16" else None
    engine, plain, without = engines8(name, dtype), Plain8(model_dirs[name], round_to=rounded), PlainGpt2(model_dirs[name], round_to=rounded)
    for n in (1, 7, 100):
        toks = random_tokens(n, n, TINY[name]["vocab_size"])
        want = plain.logits(toks)
        far = rel_err(without.logits(toks), want)
        assert rel_err(run(engine, [toks]), want) <= 2 * far, (n, far)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_whole_prompts_and_token_by_token(engines8, dtype):
    engine = engines8("D", dtype)
    toks = random_tokens(3, 150, TINY["D"]["vocab_size"])
    whole = run(engine, [toks])
    for pieces in ([[t] for t in toks], [toks[:70], toks[70:71], toks[71:]]):
        assert rel_err(run(engine, pieces), whole) <= TOL[dtype]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_unequal_prompts_together(engines8, dtype):
    engine = engines8("D", dtype)
    prompts = [random_tokens(i, n, TINY["D"]["vocab_size"]) for i, n in enumerate((1, 64, 200, 65, 3))]
    alone = [run(engine, [p])[-1] for p in prompts]
    slots = [engine.open() for _ in prompts]
    together = engine.step([StepEntry(s, p, (len(p) - 1,)) for s, p in zip(slots, prompts)]).cpu().numpy()
    for s in slots:
        engine.close(s)
    assert rel_err(together, np.stack(alone)) <= TOL[dtype]


def test_generation_is_greedy_of_its_own_logits_and_8_bits_stay_near(engines8, engines, model_dirs):
    engine = engines8("A", "bfloat16")
    prompts = [random_tokens(i, n, TINY["A"]["vocab_size"]) for i, n in enumerate((5, 11, 17))]
    outs = engine.generate(prompts, max_tokens=40, temperature=0.0)
    assert outs == engine.generate(prompts, max_tokens=40, temperature=0.0)          # (captured by now)
    for p, o in zip(prompts, outs):
        ref = run(engine, [p + o])
        for j, tok in enumerate(o):
            row = ref[len(p) - 1 + j]
            assert row.max() - row[tok] <= 2 * TOL["bfloat16"] * np.abs(row).max()
    engine.cache.book.check_all_free()
    # 8 bits a weight, an activation and a cached entry are an approximation: of the engine without them, to a few hundredths
    toks = random_tokens(1, 60, TINY["A"]["vocab_size"])
    assert 1e-4 < rel_err(run(engine, [toks]), run(engines("A", "bfloat16"), [toks])) < 0.1


def test_weights_and_cache_take_about_half(engines8, engines):
    a, b = engines8("D", "bfloat16"), engines("D", "bfloat16")
    assert a.cache.bytes() == b.cache.bytes() * (64 + 4) // (2 * 64)
    inside = lambda e: sum(t.numel() * t.element_size() for blk in e.model.blocks for t in blk.tensors() if t.dim() == 2)
    assert inside(a) * 2 == inside(b)
