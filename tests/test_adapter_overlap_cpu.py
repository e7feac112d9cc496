"""Which outputs of the adapter calls overlap what is still read."""
import pytest

from diffuser_b200 import ops


# addresses in one buffer whose rows are 128 bytes apart: out is 40 bytes wide and starts at 1000
@pytest.mark.parametrize("at,stride,width,rows,meets", [
    (1000 + 40, 128, 88, 9, False),         # the rest of the same rows
    (1000 + 40, 128, 96, 9, True),          # up to the next row's start and into it
    (1000 + 32, 128, 40, 9, True),          # a column range that starts inside
    (1000 - 32, 128, 40, 9, True),          # and one that ends inside
    (1000 - 40, 128, 40, 9, False),
    (1000 + 3 * 128 + 8, 128, 16, 2, True),  # inside, rows further down
    (1000 + 3 * 128 + 48, 128, 16, 2, False),
    (1000 + 9 * 128, 128, 40, 4, False),    # behind the last row
    (1000 + 8 * 128 + 40, 128, 40, 4, False),
    (1000 + 8 * 128 + 39, 64, 40, 4, True),  # another stride: taken by its range
    (1000 - 4 * 64, 64, 40, 4, False),
    (1000 + 64, 0, 8, 0, False),            # nothing there
])
def test_rows_that_meet_are_refused(at, stride, width, rows, meets):
    out = (1000, 128, 40, 9, "out")
    if meets:
        with pytest.raises(ValueError, match="overlap it"):
            ops._refuse_alias(out, ((at, stride, width, rows, "it"),))
    else:
        ops._refuse_alias(out, ((at, stride, width, rows, "it"),))
    ops._refuse_alias((1000, 128, 40, 0, "out"), ((at, stride, width, rows, "it"),))


def test_every_byte_of_small_layouts():
    def touched(p, ld, w, m):
        return {p + i * ld + j for i in range(m) for j in range(w)}
    for stride in (4, 6):
        for at in range(0, 30):
            for width in range(1, stride + 1):
                for rows in (1, 2, 3):
                    out, it = (10, 6, 2, 3), (at, stride, width, rows)
                    try:
                        ops._refuse_alias((*out, "out"), ((*it, "it"),))
                        free = True
                    except ValueError:
                        free = False
                    meet = bool(touched(*out) & touched(*it))
                    assert not (free and meet), it
                    # of one stride exactly, with another one by the range
                    assert free or meet or stride != 6 or rows == 1, it
