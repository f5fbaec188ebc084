"""Adapters of ranks beyond 64, whose B and t a warp takes in pieces of 64 ranks, against 64 bits: tiles of 8 and of 32 rows with one and with several units
of outputs a warp, ranks of every size in one call, and the row counts at which tiles fill up and change their size."""
import pytest
from test_gpu_adapters import Set, mixed, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,slots,rank,k,outs", [
    (1, 2, 72, 256, [14336]), (1, 1, 128, 264, [14336]), (5, 3, 200, 512, [14335, 4000]), (3, 2, 256, 136, [28672]),
    (64, 32, 128, 256, [4096, 1024, 1024]), (64, 32, 248, 72, [4096]), (48, 16, 136, 1000, [9000])])
def test_many_units_a_warp(wv, dtype, rows, slots, rank, k, outs):
    """Tiles of 8 rows: t's pieces change with every unit's pieces, from the first unit of a warp to its last."""
    s = Set(wv, dtype, slots, rank, k, outs)
    run(s, mixed(rows, slots) if rows > 1 else [slots - 1])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [36, 400])
def test_ranks_below_and_above_a_piece(wv, dtype, rows):
    """Ranks from none to 256 in one call, in tiles of 8 rows and of 32; what stands behind an adapter's rank is NaN."""
    ranks = [0, 1, 63, 64, 65, 80, 127, 128, 129, 191, 192, 193, 255, 256]
    s = Set(wv, dtype, len(ranks), 256, 200, [4099, 50], ranks=ranks)
    run(s, [i % 15 - 1 for i in range(rows)], inplace=rows == 36)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rank", [16, 40, 128])
@pytest.mark.parametrize("rows", [7, 8, 9, 31, 32, 33, 40, 64, 65])
def test_rows_of_one_adapter(wv, dtype, rank, rows):
    """Up to 8 rows of one adapter are one tile of 8, from 9 on tiles of 32."""
    run(Set(wv, dtype, 1, rank, 128, [2100]), [0] * rows)
