"""Which way a captured step of beams reads its keys, at sizes where both were measured, and what a step counts."""
import pytest

from rustinfer_b200.ops.kernels import _beam_row_tiles, attention_beams_sooner

# heads, key heads, head size, requests, beams, common keys, own keys, us a layer row by row, together
MEASURED = [
    (32, 8, 64, 4, 4, 8273, 60, 114, 104), (32, 8, 64, 4, 4, 8273, 400, 115, 115), (32, 8, 64, 8, 8, 1536, 60, 108, 109),
    (32, 8, 64, 8, 8, 4116, 150, 144, 120), (32, 8, 64, 8, 8, 4000, 1000, 155, 171), (32, 8, 64, 8, 8, 16000, 1000, 320, 197),
    (32, 8, 64, 1, 4, 33095, 10, 101, 113), (32, 8, 64, 1, 8, 16547, 60, 102, 108), (32, 8, 64, 2, 4, 16547, 60, 101, 99),
    (32, 8, 64, 24, 2, 5488, 60, 140, 145), (32, 8, 64, 24, 2, 1365, 60, 104, 107), (32, 8, 64, 16, 2, 8232, 150, 137, 128),
    (32, 8, 64, 16, 4, 4000, 600, 148, 155), (32, 8, 64, 4, 8, 2048, 800, 99, 133), (32, 8, 64, 1, 16, 8273, 60, 113, 116),
    (32, 8, 64, 1, 64, 300, 10, 90, 103), (32, 8, 128, 4, 8, 1024, 60, 164, 168), (32, 8, 128, 4, 8, 2068, 60, 180, 171),
    (32, 8, 128, 4, 8, 2068, 400, 186, 194), (32, 8, 128, 4, 8, 4116, 400, 215, 201), (32, 8, 128, 16, 4, 1034, 400, 233, 218),
    (32, 8, 128, 16, 4, 1000, 1000, 249, 256), (32, 8, 128, 12, 4, 1378, 400, 258, 219), (32, 8, 128, 1, 4, 16547, 60, 192, 190),
    (32, 8, 128, 1, 4, 16000, 1000, 192, 231), (32, 8, 128, 1, 64, 4000, 600, 315, 239), (32, 8, 128, 16, 2, 1536, 150, 173, 183),
    (32, 8, 128, 16, 2, 4116, 400, 216, 229), (32, 8, 128, 1, 16, 8232, 250, 353, 320), (24, 8, 128, 1, 8, 8273, 60, 135, 127),
    (24, 8, 128, 4, 4, 4136, 400, 164, 168), (32, 8, 128, 2, 2, 32931, 10, 219, 213),
    (32, 8, 128, 1, 4, 300, 10, 164, 168), (24, 8, 128, 8, 8, 1536, 400, 193, 168)]


@pytest.mark.parametrize("heads,kv_heads,dim,requests,beams,common,own,rows_us,together_us", MEASURED)
def test_the_way_that_is_chosen_is_the_sooner_one(heads, kv_heads, dim, requests, beams, common, own, rows_us, together_us):
    """To 4 %."""
    together = attention_beams_sooner(requests * beams, beams, heads, kv_heads, dim, requests * beams * common, own)
    assert (together_us if together else rows_us) <= 1.04 * min(rows_us, together_us)


def test_more_common_keys_or_fewer_own_ones_never_turn_it_back():
    for rows, beams, dim in ((64, 8, 64), (64, 16, 128), (32, 2, 128), (8, 4, 128), (4, 4, 64), (40, 8, 64)):
        for own in (1, 64, 300, 1000):
            chosen = [attention_beams_sooner(rows, beams, 32, 8, dim, rows * n, own) for n in range(0, 40000, 500)]
            assert chosen == sorted(chosen)
        for n in (500, 2000, 9000, 30000):
            chosen = [attention_beams_sooner(rows, beams, 32, 8, dim, rows * n, own) for own in range(1, 3000, 50)]
            assert chosen == sorted(chosen, reverse=True)


def test_row_tiles_are_the_kernels():
    from rustinfer_b200.ops import library
    lib = library.attention_beams(64)
    assert [_beam_row_tiles(n) for n in range(1, 513)] == [lib.ri_attention_beams_row_tiles(n) for n in range(1, 513)]
