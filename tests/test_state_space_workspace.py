"""How much scratch the state space scan asks for: by the tokens that are cut into blocks, not by the number of sequences (no GPU needed)."""
import ctypes

import pytest


def _bytes(**kw):
    from lampa_b200 import _lib
    n = ctypes.c_size_t(0)
    d = _lib.SsmDesc(**dict(dict(B=1, T=1000, H=16, P=64, N=128, G=1, nseq=0, dtype=0, dt_dtype=0, dt_softplus=1), **kw))
    assert _lib.lib().lampa_ssm_workspace_bytes(ctypes.byref(d), ctypes.byref(n)) == 0
    return n.value


@pytest.mark.parametrize("dtype", [0, 1])
def test_sequences_of_one_block_need_none(dtype):
    assert _bytes(B=4096, T=128, dtype=dtype) == 0
    assert _bytes(B=300, T=100, dtype=dtype) == 0
    assert _bytes(B=1, T=64, dtype=dtype) == 0


@pytest.mark.parametrize("dtype", [0, 1])
def test_a_packed_batch_does_not_pay_for_its_sequences(dtype):
    few, many = _bytes(T=655360, nseq=1, dtype=dtype), _bytes(T=655360, nseq=16384, dtype=dtype)
    assert many <= few < 200 << 20                # 2.7 GB of x


def test_slots_of_long_sequences_do_not_meet():
    """Blocks of bl tokens of every sequence of more than bl: slots floor(2 begin / bl) + block, all different and below floor(2 tokens / bl)"""
    import random
    rng = random.Random(0)
    for _ in range(300):
        bl = 64 * rng.choice([1, 2, 3, 7])
        lens = [rng.choice([0, 1, bl - 1, bl, bl + 1, 2 * bl, rng.randint(0, 9 * bl)]) for _ in range(rng.randint(1, 30))]
        taken, begin = [], 0
        for n in lens:
            if n > bl:
                taken += [begin // (bl // 2) + b for b in range(-(-n // bl))]
            begin += n
        assert len(set(taken)) == len(taken) and all(0 <= s < begin // (bl // 2) for s in taken)
