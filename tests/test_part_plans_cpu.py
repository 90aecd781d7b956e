"""Plans of attention over shared prefixes, made on the host for a device of 256 units: where
the groups' partial rows lie and what workspace a call takes."""

import json
import random
import subprocess
import sys

import pytest

from small_q_attention_amd import build

PLANNER = """
import ctypes, importlib.util, json, sys

units = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)  # found before the library's own
lib = ctypes.CDLL(sys.argv[2])
lib.sqa_shared_workspace_bytes.restype = ctypes.c_size_t
lib.sqa_last_error.restype = ctypes.c_char_p
names = json.loads(sys.argv[3])

class Plan(ctypes.Structure):
    _fields_ = [("struct_size", ctypes.c_size_t)] + [(n, ctypes.c_int) for n in names]

out = []
for groups, shape, kv, most, width in json.load(sys.stdin):
    flat = [x for g in groups for x in g]
    plan, table = Plan(), (ctypes.c_int32 * (len(flat) + 2 * shape[0]))()
    rc = lib.sqa_plan_shared_prefix(0, *shape, kv, len(groups),
                                    (ctypes.c_int32 * max(len(flat), 1))(*flat), most, width,
                                    ctypes.byref(plan), table)
    out.append({"rc": rc, "error": (lib.sqa_last_error() or b"").decode(), "table": list(table),
                "bytes": lib.sqa_shared_workspace_bytes(ctypes.byref(plan)),
                **{n: getattr(plan, n) for n in names}})
json.dump(out, sys.stdout)
"""


@pytest.fixture(scope="module")
def plans(tmp_path_factory):
    """Plans of ``(groups, (batch, q_len, query heads, kv heads, head_dim, page_size), kv_dtype,
    max_seq_len, max_pages)``, in a process that counts the device's units itself."""
    if build.is_stale():
        build.build()
    from small_q_attention_amd import _lib

    at = tmp_path_factory.mktemp("planner")
    (at / "units.c").write_text("int sqa_device_cu_count(int device) { return 256; }\n")
    subprocess.run(["gcc", "-shared", "-fPIC", "-o", str(at / "units.so"), str(at / "units.c")],
                   check=True)
    names = [n for n, _ in _lib.SharedPlan._fields_[1:]]

    def make(calls):
        res = subprocess.run([sys.executable, "-c", PLANNER, str(at / "units.so"),
                              str(build.LIB_PATH), json.dumps(names)], input=json.dumps(calls),
                             capture_output=True, text=True)
        assert res.returncode == 0, res.stderr
        return json.loads(res.stdout)

    make.units = str(at / "units.so")
    return make


def _splits(groups, plan, page):
    """Splits of each group: as many of at most shared_size pages as it takes, all alike."""
    out = []
    for _, count, pages in groups:
        pages *= page // 16 * (count > 1)
        each = -(-pages // -(-pages // plan["shared_size"])) if pages else 1
        out.append(-(-pages // each))
    return out


def _used(groups, plan, shape):
    """Slots that a call writes: a sequence's own ones and its group's splits."""
    own = plan["num_splits"] * (shape[0] if plan["pages_per_split"] else 1)
    return own + sum(count * n for (_, count, _), n in zip(groups, _splits(groups, plan, shape[5])))


def _slot_bytes(shape):
    return shape[1] * shape[2] * (shape[4] + 2) * 4


WIDE = (512, 4, 64, 8, 128, 16)
UNLIKE = [
    ([(0, 2, 8192), (2, 510, 64)], WIDE, 8192 + 64),
    ([(0, 2, 2048)] + [(2 * i, 2, 32) for i in range(1, 256)], WIDE, 2048 + 64),
    ([(0, 2, 8192)] + [(2 * i, 2, 32) for i in range(1, 512)], (1024, *WIDE[1:]), 8192 + 64),
    ([(0, 2, 8192), (2, 254, 64)], (256, 4, 32, 8, 128, 16), 8192 + 64),
    ([(510, 2, 8192)], WIDE, 8192 + 64),
    ([(0, 510, 64), (510, 2, 8192)], WIDE, 8192 + 64),
]


@pytest.mark.parametrize("groups,shape,width", UNLIKE)
@pytest.mark.parametrize("kv", [0, 2])
def test_one_long_prefix_does_not_size_the_batch(plans, groups, shape, width, kv):
    """The workspace follows what the call writes: no slot that stays empty beyond one or two
    for each sequence."""
    calls = [(groups, shape, kv, most, width) for most in (0, 16 * width)]
    for plan in plans(calls):
        assert plan["rc"] == 0, plan["error"]
        # 8 bytes of a table for each sequence where the own pages are cut across sequence ends.
        most = (_used(groups, plan, shape) + 2 * shape[0]) * _slot_bytes(shape) + 8 * shape[0]
        assert plan["bytes"] <= most
        assert plan["bytes"] < 2 << 30


def test_slots_of_all_sequences_are_apart(plans):
    """Drawn groups: the slots that the plan's table and size give, as the kernels find them."""
    rng = random.Random(11)
    calls = []
    for i in range(400):
        batch, page = rng.randint(2, 300), rng.choice([16, 64, 256])
        groups, at = [], 0
        while at < batch:
            count = min(rng.choice([1, 2, 2, 3, rng.randint(1, batch)]), batch - at)
            pages = rng.choice([0, 1, 2, rng.randint(1, 40), rng.randint(1, 40), 3000 * 16 // page])
            if rng.random() < 0.8:
                groups.append((at, count, pages))
            at += count
        width = max([p for *_, p in groups] + [1]) + rng.randint(1, 20)
        d = rng.choice([64, 128, 256])
        calls.append((groups, (batch, rng.randint(1, 4), 8, rng.choice([1, 2, 8]), d, page),
                      rng.choice([0, 2]), 0, width))
    calls = [c for c in calls if c[1][1] * (8 // c[1][3]) <= (32 if c[1][4] == 256 else 64)]
    packed = 0
    for (groups, shape, *_), plan in zip(calls, plans(calls)):
        assert plan["rc"] == 0, plan["error"]
        splits, size = _splits(groups, plan, shape[5]), plan["shared_size"]
        if not plan["num_items"]:
            continue
        is_packed = plan["shared_splits"] < max(splits)
        packed += is_packed
        of = plan["table"][3 * len(groups):]
        used = set()
        for (first, count, pages), n in zip(groups, splits):
            for b in range(first, first + count):
                before, own = of[2 * b:2 * b + 2]
                if n == 0:
                    assert before == -1
                    continue
                assert own == pages
                mine = ({b + before // size + j for j in range(n)} if is_packed
                        else {b + j * shape[0] for j in range(n)})
                assert not used & mine
                used |= mine
        assert max(used) < plan["shared_splits"] * shape[0]
    assert packed > 20


def test_plans_of_huge_batches_keep_to_a_few_gib(plans):
    """Thousands of sequences over long tables: cuts into many splits, whose partial rows take
    tens of GB, are left for others; what a batch cannot do without (a row of its own and one of
    its group's each) is not refused."""
    rng = random.Random(3)
    calls = []
    for _ in range(300):
        batch = rng.choice([1000, 3000, 8192])
        hkv, d = rng.choice([1, 8, 16]), rng.choice([64, 128, 256])
        hq = hkv * rng.choice([1, 4, 8])
        q = rng.randint(1, (32 if d == 256 else 64) // (hq // hkv))
        width, groups, at = rng.choice([500, 8000, 150000]), [], 0
        for _ in range(rng.choice([1, 3, 40])):
            count = min(rng.choice([2, 3, 600, 8192]), batch - at)
            if count > 0:
                groups.append((at, count, rng.randint(1, width)))
            at += count
        calls.append((groups, (batch, q, hq, hkv, d, 16), 0, rng.choice([0, 16 * width]), width))
    for (groups, shape, *_, width), plan in zip(calls, plans(calls)):
        assert plan["rc"] == 0, plan["error"]
        least = 3 * shape[0] * _slot_bytes(shape)
        assert plan["bytes"] <= max(5 << 30, least + 8 * shape[0])


def test_cuts_of_windows_keep_to_a_few_gib(plans):
    script = """
import ctypes, json, sys
units = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
lib = ctypes.CDLL(sys.argv[2])
lib.sqa_workspace_bytes.restype = ctypes.c_size_t
n = [ctypes.c_int() for _ in range(3)]
for batch, q, hq, hkv, d, window, width in json.load(sys.stdin):
    assert lib.sqa_plan_windowed(0, batch, q, hq, hkv, d, ctypes.c_int64(window), 4, 0, width, 0,
                                 *(ctypes.byref(x) for x in n)) == 0
    assert lib.sqa_workspace_bytes(batch, q, hq, hkv, d, n[0].value, n[1].value) < 5 << 30
"""
    rng = random.Random(4)
    calls = [(rng.choice([1300, 2000, 4464]), 8 // g, 16 * g, 16, d, rng.choice([900000, 10**6]),
              rng.choice([96000, 180000])) for g in (1, 4, 8) for d in (64, 128) for _ in range(8)]
    calls.append((1937, 8, 128, 16, 128, 1044825, 95985))
    res = subprocess.run([sys.executable, "-c", script, plans.units, str(build.LIB_PATH)],
                         input=json.dumps(calls), capture_output=True, text=True)
    assert res.returncode == 0, res.stderr
