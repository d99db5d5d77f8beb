"""How flash_decode runs a call (csrc/decode_plan.h): what has to hold whatever the borders are. No GPU."""
import random

from decode_plans import plan


def test_plans_cover_the_rows_and_fit_the_kernels():
    rng = random.Random(1)
    seen = set()
    for _ in range(4000):
        kv_heads, group, tokens = rng.randint(1, 16), rng.randint(1, 32), rng.choice([1, 1, 2, 3, 8, 40, 500, 2048])
        batch, room = rng.choice([1, 2, 7, 32, 500]), 8 * rng.randint(1, 20000)
        head_dim, window = rng.choice([64, 128]), rng.choice([-1, -1, 0, 5, 300, 4000, 2 ** 31 - 1])
        d = plan(batch, tokens, group * kv_heads, kv_heads, room, head_dim, window)
        rows = group * tokens
        assert (d.row_tiles - 1) * d.part_rows < rows <= d.row_tiles * d.part_rows
        assert d.items == batch * kv_heads * d.row_tiles
        # rows of a CTA of the kernel that is launched: decode_kernel's by part_rows, decode_wide_kernel 128
        assert d.part_rows in ((32, 64, 128) if d.wide else (16, 32, 64))
        assert not d.wide or d.part_rows == 128 or d.row_tiles == 1
        assert d.cluster in ((0, 1) if d.wide else (0, 1, 4, 8))
        # every key that a row tile may see lies in its tiles
        keys = 64 if head_dim == 128 else 128
        assert d.tiles * keys >= min(room, window + tokens + keys - 1 if window >= 0 else room)
        seen.add((d.wide, d.part_rows, d.cluster))
    assert {(w, r, c) for w, r, c in seen if w} >= {(1, 32, 0), (1, 64, 0), (1, 128, 0), (1, 128, 1)}
    assert {c for w, r, c in seen if not w} == {0, 1, 4, 8}
