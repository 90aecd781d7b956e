"""Random shapes, types, lengths and masks through the operators around the paged cache,
each against its plain statement in 64 bits."""

import math
import random

import pytest

torch = pytest.importorskip("torch")

from tests import test_gpu_eviction as ev  # noqa: E402
from tests import test_gpu_scaled_cache as sc  # noqa: E402

pytestmark = pytest.mark.gpu

E4M3, INT8, F16, BF16 = torch.float8_e4m3fn, torch.int8, torch.float16, torch.bfloat16


def _shape(rng, most_tokens):
    hkv, group = rng.choice([1, 2, 3, 4, 5, 8, 9]), rng.choice([1, 2, 4, 5, 8])
    d, page = rng.choice([64, 128, 128, 256]), rng.choice([16, 16, 32, 64, 128, 256])
    batch = rng.choice([1, 1, 2, 3, 7, 20])
    top = max(2, int(math.exp(rng.uniform(0.7, math.log(most_tokens / batch)))))
    lens = [rng.choice([0, 1, rng.randint(0, top), rng.randint(0, top), top,
                        max(1, top // page * page)]) for _ in range(batch)]
    q_len = rng.randint(1, max(1, min(17, (32 if d == 256 else 64) // group)))
    return hkv, group, d, page, lens, q_len


@pytest.mark.parametrize("seed", range(40))
def test_attention(seed):
    rng = random.Random(1000 + seed)
    hkv, group, d, page, lens, q_len = _shape(rng, 6000)
    trees = sc._trees(len(lens), q_len, seed, (rng.randint(0, q_len),)) if rng.random() < 0.4 \
        else None
    sc._check(lens, q_len, hkv * group, hkv, d, page, rng.choice([F16, BF16]),
              rng.choice([E4M3, INT8]), seed=seed, trees=trees,
              width=max(1, -(-max(lens) // page)) + rng.choice([0, 0, 1, 30]))


@pytest.mark.parametrize("seed", range(40))
def test_weights(seed):
    rng = random.Random(2000 + seed)
    hkv, group, d, page, lens, q_len = _shape(rng, 6000)
    trees = sc._trees(len(lens), q_len, seed, (rng.randint(0, q_len),)) if rng.random() < 0.4 \
        else None
    ev._check_weigh(lens, q_len, hkv * group, hkv, d, page, rng.choice(ev.TYPES), seed=seed,
                    trees=trees, cut=rng.choice([0, 0, 1, 37]),
                    width=max(1, -(-max(lens) // page)) + rng.choice([0, 0, 1, 30]))


@pytest.mark.parametrize("seed", range(30))
def test_append(seed):
    rng = random.Random(3000 + seed)
    hkv, _, d, page, lens, _ = _shape(rng, 1500)
    q_len = rng.choice([1, 2, 5, 16, rng.randint(1, 300)])
    new = None if rng.random() < 0.3 else [rng.randint(0, q_len + 1) for _ in lens]
    sc._check_append(*sc._append_case(lens, new, q_len, hkv, d, page, rng.choice([F16, BF16]),
                                      rng.choice([E4M3, INT8]), seed=seed))


@pytest.mark.parametrize("seed", range(30))
def test_evict(seed):
    rng = random.Random(4000 + seed)
    hkv, _, d, page, lens, _ = _shape(rng, 3000)
    budget = rng.choice([1, 15, 16, 17, 64, max(1, max(lens) // 2), max(lens) + 3])
    sink = rng.choice([0, 0, min(4, budget), budget])
    recent = rng.choice([0, (budget - sink) // 2, budget - sink])
    ev._check_evict(ev._evict_case(lens, hkv, d, page, rng.choice(ev.KINDS), budget, seed=seed,
                                   ties=rng.random() < 0.5),
                    budget, sink, recent, in_place=rng.random() < 0.5 and budget <= max(lens))
