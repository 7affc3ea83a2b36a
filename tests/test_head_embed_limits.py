"""Refusals of sizes past what the kernels' launches and whole numbers hold, without a GPU."""
import pytest

from test_head_embed import run_c


@pytest.mark.parametrize("body", [
    "head(x=t(1000000001, 1), targets=t(1000000001), W=t(3, 1))",
    "head(x=t(2147483647, 1), targets=t(2147483647), W=t(3, 1), dx=t(2147483647, 1), dW=t(3, 1))"])
def test_too_many_rows(body):
    """Rows go through in pieces, and the place behind the last piece has to fit a whole number."""
    r = run_c(body)
    assert r.returncode == 1 and "survived" not in r.stdout and "up to 1000000000 rows" in r.stderr, r.stderr


def test_as_many_rows_as_there_may_be():
    """Gets as far as the runtime, which is not up."""
    r = run_c("head(x=t(1000000000, 1), targets=t(1000000000), W=t(3, 1))")
    assert r.returncode == 1 and "runtime_init" in r.stderr, r.stderr
