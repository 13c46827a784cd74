"""More of what the paged cache's C entry points refuse before any launch; these run without a GPU."""
import pytest

from tests.test_paged_cpu import A, lib, refused  # noqa: F401  (lib is a fixture)


def test_negative_strides(lib):
    """Offsets below zero stand for rows that are not there."""
    S = lib.Strides3
    row, pages = S(0, 64, 256), S(2048, 1024, 64)
    ok = [A, A, A, A + 4096, row, pages, row, A, A, A, 2, 8, 3, 1, 4, 2, 64, 16, 8, 0.125, lib.BF16]
    for at, bad in [(4, S(0, -64, 256)), (4, S(0, 64, -256)), (6, S(0, -64, 256)), (6, S(0, 64, -256)), (5, S(-2048, 1024, 64)),
                    (5, S(2048, -1024, 64)), (5, S(2048, 1024, -64))]:
        refused(lib.attn_paged, [bad if i == at else v for i, v in enumerate(ok)], "negative", lib)
    st = S(0, 64, 128)
    ok = [A, A, A, A, st, st, pages, A, 3, 2, 64, 16, 8, lib.F16]
    for bad in (S(-2048, 1024, 64), S(2048, -1024, 64), S(2048, 1024, -64)):
        refused(lib.paged_append, [bad if i == 6 else v for i, v in enumerate(ok)], "negative", lib)
