"""How the paged attention deals its work to workgroups, on the CPU: the kernels' own plan functions compiled for the host
(paged_plan_host.hip). Every place of a plan has a workgroup, and every part that is joined a slot of the workspace."""
import ctypes
import math
import os
import random
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope='module')
def plan(tmp_path_factory):
    from streamvoxel_amd.build import hipcc
    path = str(tmp_path_factory.mktemp('plan') / 'libplan.so')
    res = subprocess.run([hipcc(), '-O2', '-std=c++17', '-fPIC', '-shared', '--offload-host-only',
                          os.path.join(HERE, 'paged_plan_host.hip'), '-o', path], capture_output=True)
    assert res.returncode == 0, res.stderr.decode()
    fn = ctypes.CDLL(path).plan_places
    fn.restype = None
    fn.argtypes = [ctypes.c_int64] * 4 + [ctypes.c_void_p] * 2 + [ctypes.c_int64] * 3 + [ctypes.c_int, ctypes.c_void_p]

    def call(counts, lengths, H, Hkv, page=64, D=64, fp8=False, packed=True):
        """counts: tokens of every window (packed), or of each."""
        B = len(lengths)
        cu = None
        if packed:
            cu = (ctypes.c_int32 * (B + 1))(*[sum(counts[:b]) for b in range(B + 1)])
        held, out = (ctypes.c_int32 * B)(*lengths), (ctypes.c_int64 * 9)()
        fn(B, H, Hkv, sum(counts) if packed else counts[0], cu, held, D, max(1, -(-max(lengths) // page)), page, fp8, out)
        return dict(zip(('places', 'grid', 'lost', 'slots_used', 'slots', 'rows', 'row_grid', 'row_slots_used', 'row_slots'),
                        out))

    def check(*args, **kw):
        p = call(*args, **kw)
        assert p['lost'] == 0 and p['places'] <= p['grid'], p
        assert p['slots_used'] <= p['slots'], p
        assert p['rows'] <= p['row_grid'] and p['row_slots_used'] <= p['row_slots'], p
        return p
    return check


@pytest.mark.parametrize('fp8, n', [(False, 5), (True, 17)])
@pytest.mark.parametrize('times', [1, 2])
def test_a_long_window_among_tiles_beside_single_tokens(plan, times, fp8, n):
    """Tiles that fill the half of the chip that they have beside single tokens, and one window cut for all that: more places
    than the chip's full share."""
    counts = [n] * 52 * times + [1] * 8 * times
    lengths = [64000] + [384] * (52 * times - 1) + [8192] * 8 * times
    p = plan(counts, lengths, 8 // times, 8 // times, fp8=fp8, D=16)
    assert p['places'] > 512 and p['slots_used'] > 0


def test_plans_of_random_calls(plan):
    rng = random.Random(4)
    log = lambda low, high: int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    cut = beside = 0
    for _ in range(4000):
        B, Hkv, G, fp8 = log(1, 300), rng.choice([1, 2, 4, 8, 16]), rng.choice([1, 1, 2, 4]), rng.random() < 0.3
        tokens = log(1, 500)
        counts = [rng.choice([0, 1, 1, rng.randint(1, tokens), tokens]) for _ in range(B)]
        counts[0] = max(counts[0], 1)
        short, long = log(1, 4000), log(1, 100000)
        lengths = [long if rng.random() < 0.05 else rng.randint(0, short) for _ in range(B)]
        packed = rng.random() < 0.7
        if not packed:
            counts = [tokens] * B
        p = plan(counts, lengths, G * Hkv, Hkv, rng.choice([16, 64, 256]), fp8=fp8, packed=packed)
        cut += p['slots_used'] > 0
        beside += p['places'] > 0 and p['rows'] > 0
    assert cut > 300 and beside > 300
