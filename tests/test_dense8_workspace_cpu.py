"""The workspace of inf_linear_int belongs to the kernel that the call takes."""
import pytest


def size(*args):
    from inf_hip import lib
    return lib.inf_linear_int_call_workspace_bytes(*args)


@pytest.mark.parametrize("rows,n,k", [(1, 1, 1), (16, 256, 1024), (17, 300, 40), (16383, 256, 256), (16384, 256, 256),
                                      (16384, 32, 256), (16384, 33, 1), (40000, 256, 257), (40000, 257, 256),
                                      (262144, 256, 1024), (1 << 30, 40, 24)])
def test_enough_for_any_call(rows, n, k):
    """Never more than the size for any act and add; the form that holds the weight in LDS (16,384 rows and more,
    k <= 256, 33 to 256 outputs, no sigmoid, nothing to add) and those that put x into 8 bits themselves need none."""
    from inf_hip import lib
    for x in (0, 1, 4):
        for out in (0, 1, 4):
            most = lib.inf_linear_int_workspace_bytes(rows, n, k, x, out)
            for act in (0, 1, 2):
                for add in (0, 1):
                    got = size(rows, n, k, x, out, act, add)
                    walks = rows >= 16384 and k <= 256 and 33 <= n <= 256 and act != 2 and not add
                    assert got == (0 if walks else most) and most >= 0


def test_refused_sizes():
    assert size(-1, 1, 1, 0, 0, 0, 0) == -1 and size(1, 0, 1, 0, 0, 0, 0) == -1 and size(1, 1, 0, 0, 0, 0, 0) == -1
