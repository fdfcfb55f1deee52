"""How attention through a sliding window deals its work to workgroups, on the CPU: the kernels' own plan functions compiled
for the host (paged_window_plan_host.hip). Every place has a workgroup, every part that is joined a slot of the workspace that
the call without a window asks for, and no tile walks more blocks than its window's parts hold."""
import ctypes
import math
import os
import random
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
NAMES = ('places', 'grid', 'lost', 'slots_used', 'slots', 'rows', 'row_grid', 'row_slots_used', 'row_slots', 'more_bytes',
         'long_tiles', 'lost_keys')


@pytest.fixture(scope='module')
def plan(tmp_path_factory):
    from streamvoxel_amd.build import hipcc
    path = str(tmp_path_factory.mktemp('plan') / 'libplan.so')
    res = subprocess.run([hipcc(), '-O2', '-std=c++17', '-fPIC', '-shared', '--offload-host-only',
                          os.path.join(HERE, 'paged_window_plan_host.hip'), '-o', path], capture_output=True)
    assert res.returncode == 0, res.stderr.decode()
    fn = ctypes.CDLL(path).window_places
    fn.restype = None
    fn.argtypes = [ctypes.c_int64] * 4 + [ctypes.c_void_p] * 2 + [ctypes.c_int64] * 3 + [ctypes.c_int] + [
        ctypes.c_int64] * 2 + [ctypes.c_void_p]

    def check(counts, lengths, H, Hkv, window, sinks, page=64, D=64, codes=False, packed=True, short=0):
        B = len(lengths)
        cu = None
        if packed:
            cu = (ctypes.c_int32 * (B + 1))(*[sum(counts[:b]) for b in range(B + 1)])
        held, out = (ctypes.c_int32 * B)(*lengths), (ctypes.c_int64 * 12)()
        pages = max(1, -(-max(lengths) // page) - short)
        fn(B, H, Hkv, sum(counts) if packed else counts[0], cu, held, D, pages, page, codes, window, sinks, out)
        p = dict(zip(NAMES, out))
        assert p['lost'] == 0 and p['places'] <= p['grid'], p
        assert p['slots_used'] <= p['slots'], p
        assert p['rows'] <= p['row_grid'] and p['row_slots_used'] <= p['row_slots'], p
        assert p['more_bytes'] == p['long_tiles'] == p['lost_keys'] == 0, p
        return p
    return check


def test_plans_of_random_calls(plan):
    rng = random.Random(6)
    log = lambda low, high: int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    cut = [0, 0]
    for _ in range(2500):
        B, packed, Hkv, G = log(1, 90), rng.random() < 0.6, rng.choice([1, 2, 3, 8]), rng.choice([1, 1, 2, 4, 7, 16])
        high = log(1, 600)
        counts = [1 if rng.random() < 0.5 else rng.randint(0, high) for _ in range(B)] if packed else [high] * B
        if sum(counts) == 0:
            counts[0] = 1
        lengths = [max(0, n + log(1, 6000) - rng.choice([1, 1, 50])) for n in counts]
        if rng.random() < 0.3:
            lengths[rng.randrange(B)] = log(6000, 60000)
        p = plan(counts, lengths, Hkv * G, Hkv, log(1, 8000), rng.choice([0, 1, 4, log(5, 500)]), page=rng.choice([16, 64, 256]),
                 D=rng.choice([16, 64, 128]), codes=rng.random() < 0.5, packed=packed, short=rng.choice([0, 0, 1, 5]))
        cut[0] += p['slots_used'] > 0
        cut[1] += p['row_slots_used'] > 0
    assert min(cut) > 100


@pytest.mark.parametrize('window, sinks', [(1, 0), (1 << 30, 1 << 30), (1 << 30, 0), (1, 1 << 30)])
def test_the_longest_windows(plan, window, sinks):
    plan([1, 300], [5000, 5000], 8, 2, window, sinks)
    plan([5], [70000], 4, 1, window, sinks, packed=False)
