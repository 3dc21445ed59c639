"""Where the Python mirror does not ask for the size of the 4-bit token step's
workspace, the library needs none."""
import random

import sparsewavecomp_amd as sw


def test_no_workspace_where_none_is_asked_for():
    need = sw.load_library().sw_window_attention_decode_fp4_workspace_bytes
    rng, most = random.Random(2), sw._FP4_WHOLE
    asked = 0
    for _ in range(4000):
        sequences = rng.choice((1, 2, 7, 64, 300, 4096, 5000))
        key_heads = rng.choice((1, 2, 8, 128, 1024))
        heads = key_heads * rng.choice((1, 3, 8, 40))
        d = rng.choice((32, 64, 96, 128))
        size = rng.choice((1, 16, 24, most - 1, most))
        width = rng.randint(1, most // size)
        assert need(sequences, size, width, heads, key_heads, d,
                    rng.choice((1, most, 10 ** 9)), rng.choice((0, 10 ** 9))) == 0
        sinks = rng.randint(0, most - 1)
        window = rng.randint(1, most - sinks)
        far = sequences, 1 << 16, 1 << 4, heads, key_heads, d
        assert need(*far, window, sinks) == 0
        asked += need(*far, most + 1 - sinks, sinks) > 0
    assert asked > 0
