"""The cross entropy without logits and the sorted gradient at sizes on either side of where their kernels change, with
the references, inputs and tolerances of test_head_loss_gpu.py and test_embed_sorted_gpu.py.

W is read as it comes for few rows, up to 4096: as a multiple of 128, up to 256 + min(900, room), room = 1.4e9 /
(V (C + 100)), or for the loss alone 600 + room; for small tables, of a room past 8192, always; else it is laid out first; there are kernels for 32, 64 and 128 rows at once, and the gradient of W has its own up to 128 rows.  Up to 1024 ids are compared with each
other; the sort ranks up to 12288 rows, then goes by digits, with more rows a workgroup from 131073 on; rows that are to be overwritten are not cleared where
min(n, V) C >= 2^23.
"""
import numpy as np
import pytest

import test_embed_sorted_gpu as sorted_gpu
import test_head_loss_gpu as head

pytestmark = pytest.mark.gpu

MANY = 4225  # rows past 4096: W is laid out


@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("R,V,C", [
    (4096, 130, 36), (4097, 1, 1), (4097, 2, 3), (4100, 129, 33), (4225, 257, 100), (4351, 127, 65), (5000, 700, 64),
    (8193, 300, 31), (900, 3001, 336), (16384, 140, 16)])
def test_many_rows(rt, R, V, C, weights):
    a = head.inputs(R, V, C, weights=weights)
    ref = head.Exact(*a)
    head.agree(head.Call(rt, *a), ref)
    head.agree(head.Call(rt, *a, dx=False, dW=False), ref)


@pytest.mark.parametrize("V,C", [(127, 31), (257, 32), (300, 33), (129, 96), (1000, 130)])
@pytest.mark.parametrize("R", [31, 32, 33, 64, 65, 96, 127, 128, 129, 255, 385])
def test_few_rows(rt, R, V, C):
    a = head.inputs(R, V, C, seed=1, weights=R % 2 == 1)
    ref = head.Exact(*a)
    head.agree(head.Call(rt, *a), ref)
    head.agree(head.Call(rt, *a, dx=False, dW=False), ref)


@pytest.mark.parametrize("R", [857, 858])
def test_where_w_is_laid_out(rt, R):
    a = head.inputs(R, 50257, 20, weights=True)
    head.agree(head.Call(rt, *a), head.Exact(*a))


def test_many_rows_alike(rt):
    """The cases that may go wrong at any number of rows, at one of many."""
    head.test_parts_of_the_results(rt, MANY, 300, 40)
    head.test_padding_rows_take_no_part(rt, MANY, 200, 64)
    head.test_all_rows_padding(rt, MANY)
    head.test_targets_outside_the_vocabulary(rt, MANY)
    head.test_confident_and_far_logits(rt, MANY)
    head.test_zeros(rt, MANY)
    head.test_tensors_off_16_bytes(rt, MANY, 257, 33)
    head.test_tensors_off_16_bytes(rt, MANY, 128, 64)
    head.test_the_same_every_time(rt, MANY, 500, 80)


@pytest.mark.parametrize("shift", [-60, -30, 30, 50])
def test_many_rows_far_from_one(rt, shift):
    head.test_values_far_from_one(rt, MANY, shift)


def test_many_rows_of_other_sizes(rt):
    head.test_rows_and_columns_of_other_sizes(rt, MANY)


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_many_rows_not_finite(rt, bad):
    head.test_values_that_are_not_finite(rt, MANY, bad)


def test_many_rows_against_differences(rt):
    head.test_gradients_against_differences(rt, MANY)


@pytest.mark.parametrize("R", [32, 64, 128, 129])
def test_few_rows_alike(rt, R):
    head.test_parts_of_the_results(rt, R, 300, 40)
    head.test_padding_rows_take_no_part(rt, R, 200, 64)
    head.test_all_rows_padding(rt, R)
    head.test_targets_outside_the_vocabulary(rt, R)
    head.test_confident_and_far_logits(rt, R)
    head.test_zeros(rt, R)
    head.test_tensors_off_16_bytes(rt, R, 257, 33)
    head.test_values_that_are_not_finite(rt, R, np.nan)


@pytest.mark.parametrize("accumulate", [0, 1])
@pytest.mark.parametrize("shape,V,C,kind", [
    ((16, 1024), 9000, 936, "text"), ((13, 1000), 8200, 1028, "one"), ((13, 1000), 8200, 1027, "uniform"),
    ((13, 1000), 8193, 1024, "outside"), ((130, 1024), 300, 8, "text"), ((128, 1024), 300, 8, "text"),
    ((1, 131073), 70000, 4, "uniform"), ((20, 10000), 200000, 44, "outside"), ((300, 1000), 5, 3, "two")])
def test_sorted_gradient(rt, shape, V, C, kind, accumulate):
    sorted_gpu.test_gradient(rt, shape, V, C, kind, accumulate)


@pytest.mark.parametrize("accumulate", [0, 1])
@pytest.mark.parametrize("shape,V,C,kind", [
    ((63,), 9, 3, "two"), ((1, 64), 5, 4, "one"), ((5, 13), 8193, 5, "outside"), ((255, 1), 16385, 33, "text"),
    ((2, 128), 33, 257, "uniform"), ((257, 1), 100, 260, "one"), ((4, 256), 3, 520, "two"), ((2, 512), 5000, 36, "text"),
    ((1023, 1), 1, 7, "one"), ((32, 32), 4000000, 1, "outside"), ((1, 1025), 64, 12, "text"), ((25, 41), 2, 5, "two")])
def test_gradient_of_few_rows(rt, shape, V, C, kind, accumulate):
    sorted_gpu.test_gradient(rt, shape, V, C, kind, accumulate)


def test_few_rows_are_added_in_their_order(rt):
    sorted_gpu.test_the_same_every_time(rt, (4, 250), 90, 64, "text")
    sorted_gpu.test_the_same_every_time(rt, (1, 1024), 3, 300, "two")


@pytest.mark.parametrize("R", [438, 439, 857, 858])
def test_where_w_is_laid_out_for_gradients(rt, R):
    a = head.inputs(R, 50257, 20, seed=2, weights=True)
    ref = head.Exact(*a)
    head.agree(head.Call(rt, *a), ref)
    head.agree(head.Call(rt, *a, dx=False), ref)
    head.agree(head.Call(rt, *a, dW=False), ref)
    head.agree(head.Call(rt, *a, dx=False, dW=False), ref)


@pytest.mark.parametrize("R,V,C", [(4129, 129, 65), (5120, 384, 1), (4097, 20, 700), (4300, 1000, 129), (12345, 64, 64)])
def test_many_rows_by_their_parts(rt, R, V, C):
    """Each gradient alone."""
    a = head.inputs(R, V, C, seed=3, weights=True)
    ref = head.Exact(*a)
    head.agree(head.Call(rt, *a, dx=False), ref)
    head.agree(head.Call(rt, *a, dW=False), ref)


@pytest.mark.parametrize("R", [40, MANY])
def test_quiet_rows_and_features_of_w(rt, R):
    """Rows and features of W of many sizes.  For dx, W's values are held to 2^-40 of the largest of all: each share's
    product with one is off by that, and so is each logit's."""
    x, W, t, w = head.inputs(R, 500, 70, weights=True)
    rng = np.random.default_rng(11)
    W = (W * np.ldexp(1.0, rng.integers(-14, 1, (500, 1))) * np.ldexp(1.0, rng.integers(-14, 1, 70))).astype(np.float32)
    W[7] = 0
    W[:, 5] = 0
    ref, got = head.Exact(x, W, t, w), head.Call(rt, x, W, t, w)
    live = head.dev(np.where(w != 0, 1.0, 0.0))[:, None]
    ad, f = ref.d.abs().sum(1)[:, None], (head.dev(w) / R).abs()[:, None]
    top = float(np.abs(W).max())
    # A logit is off by 2^-39 of `top` times its row's magnitudes more, a share by its value times twice that.
    logit = head.END * top * head.dev(np.abs(x)).sum(1)
    assert 4 * logit.max().item() < 1e-6
    ref.losses_tol = ref.losses_tol + 2 * logit * live[:, 0]
    ref.loss_tol = ref.loss_tol + (2 * logit * head.dev(np.abs(w))).sum() / R
    share = 4 * logit[:, None] * f * live
    ref.dx_tol = ref.dx_tol + head.END * top * ad + share * head.dev(np.abs(W)).amax(0)
    ref.dW_tol = ref.dW_tol + (share * head.dev(np.abs(x))).amax(0)
    head.agree(got, ref)
    assert not got.dx[:, 5].any()


def test_millions_of_rows(rt):
    """Launches whose workgroups pass 65535 in one direction, and four pieces of rows."""
    a = head.inputs(4200000, 3, 2, weights=True)
    ref = head.Exact(*a)
    head.agree(head.Call(rt, *a), ref)
    head.agree(head.Call(rt, *a, dx=False, dW=False), ref)


@pytest.mark.parametrize("n", [40, 3000])
@pytest.mark.parametrize("accumulate", [0, 1])
def test_more_positions_than_the_ids_have(rt, n, accumulate):
    """A table of positions far longer than the sequences: the rest is zero, or left as it was."""
    rng = np.random.default_rng(6)
    g = rng.standard_normal((2, n, 3)).astype(np.float32)
    ids = sorted_gpu.ids_of("uniform", (2, n), 50)
    before = rng.standard_normal((300000, 3)).astype(np.float32)
    _, dP = sorted_gpu.gather(rt, g, ids, 1.0, np.zeros((50, 3), np.float32), before, accumulate)
    want = g.astype(np.float64).sum(0) + (before[:n] if accumulate else 0)
    tol = 3 * sorted_gpu.U * (np.abs(g).sum(0) + np.abs(before[:n]))
    sorted_gpu.close("dP", dP[:n], want, tol)
    assert np.array_equal(dP[n:], before[n:] if accumulate else np.zeros_like(before[n:]))


@pytest.mark.parametrize("R", [640, 641, 1152, 1153])
def test_where_w_is_laid_out_by_128_rows(rt, R):
    a = head.inputs(R, 50257, 20, seed=4, weights=True)
    ref = head.Exact(*a)
    head.agree(head.Call(rt, *a), ref)
    head.agree(head.Call(rt, *a, dx=False, dW=False), ref)


@pytest.mark.parametrize("R,V,C", [(3, 300, 1024), (5, 200, 1028), (33, 130, 2052), (65, 257, 1027), (130, 500, 1300)])
def test_few_rows_of_many_features(rt, R, V, C):
    """Rows of x that do not fit a wave's registers."""
    a = head.inputs(R, V, C, seed=5, weights=True)
    ref = head.Exact(*a)
    head.agree(head.Call(rt, *a), ref)
    head.agree(head.Call(rt, *a, dx=False, dW=False), ref)


@pytest.mark.parametrize("R", [7, 90])
def test_few_rows_where_w_changes_size(rt, R):
    """Steps of 32 tokens, and of 32 features, whose largest values are far apart: each has a scale of its own."""
    x, W, t, w = head.inputs(R, 900, 200, weights=True)
    rng = np.random.default_rng(12)
    W = (W * np.ldexp(1.0, rng.integers(-20, 1, (29, 1))).repeat(32, 0)[:900]).astype(np.float32)
    W[64:96] = 0
    W[200:232, 32:64] = 1e-38
    a = x, W, t, w
    head.agree(head.Call(rt, *a), head.Exact(*a))


@pytest.mark.parametrize("accumulate", [0, 1])
@pytest.mark.parametrize("shape,V,C,kind", [
    ((5, 8), 700, 127, "uniform"), ((5, 8), 700, 129, "uniform"), ((3, 50), 900, 130, "text"), ((1, 9), 400, 131, "two"),
    ((2, 88), 5000, 346, "outside"), ((8, 8), 300, 1601, "uniform")])
def test_rows_cleared_by_16_bytes(rt, shape, V, C, kind, accumulate):
    sorted_gpu.test_gradient(rt, shape, V, C, kind, accumulate)


@pytest.mark.parametrize("R,V,C", [(65, 129, 40), (128, 3000, 40), (300, 4700, 33), (450, 2029, 182), (512, 900, 64)])
def test_few_workgroups(rt, R, V, C):
    """Where there are few tokens, fewer rows share a reading of W."""
    a = head.inputs(R, V, C, seed=6, weights=True)
    ref = head.Exact(*a)
    head.agree(head.Call(rt, *a), ref)
    head.agree(head.Call(rt, *a, dx=False, dW=False), ref)


@pytest.mark.parametrize("R", [3, 40, 100, MANY])
@pytest.mark.parametrize("first,last", [(0, 300), (128, 256), (256, 300), (295, 296)])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_w_that_is_not_finite(rt, R, first, last, bad):
    """Any such value makes the loss NaN, whole parts of them too."""
    x, W, t, _ = head.inputs(R, 300, 40, seed=7)
    W[first:last] = bad
    for kw in ({}, {"dx": False, "dW": False}):
        got = head.Call(rt, x, W, t, **kw)
        assert np.isnan(got.loss[0]) and np.isnan(got.losses).all()


@pytest.mark.parametrize("R,V,C", [(1, 4194303, 1), (130, 1000003, 5), (400, 600001, 3)])
def test_large_vocabularies(rt, R, V, C):
    a = head.inputs(R, V, C, weights=True)
    ref = head.Exact(*a)
    head.agree(head.Call(rt, *a), ref)
    head.agree(head.Call(rt, *a, dx=False, dW=False), ref)


@pytest.mark.parametrize("accumulate", [0, 1])
@pytest.mark.parametrize("shape,V,C,kind", [
    ((7, 9), 65536, 4, "uniform"), ((7, 9), 65537, 4, "uniform"), ((1, 40), 140001, 5, "outside"), ((64,), 70000, 2, "text"),
    ((3, 5), 66000, 17, "two"), ((1, 1000), 131073, 8, "text")])
def test_rows_cleared_of_long_tables(rt, shape, V, C, kind, accumulate):
    """Ids are marked for 65536 rows at a time."""
    sorted_gpu.test_gradient(rt, shape, V, C, kind, accumulate)


@pytest.mark.parametrize("R,V,C", [(2, 50257, 45), (1, 4096, 1), (5, 4100, 129), (31, 12000, 64), (70, 9000, 200)])
def test_many_slices(rt, R, V, C):
    """The gradient of x of few rows comes in up to 512 parts."""
    a = head.inputs(R, V, C, seed=8, weights=True)
    ref = head.Exact(*a)
    one = head.Call(rt, *a)
    head.agree(one, ref)
    two = head.Call(rt, *a)
    assert np.array_equal(one.dx, two.dx)


@pytest.mark.parametrize("R,V,C", [(4100, 200, 767), (4100, 130, 768), (4097, 129, 769), (4200, 70, 1664), (4100, 100, 1665),
                                   (4099, 65, 2049)])
def test_many_rows_of_many_features(rt, R, V, C):
    """Rows of W that stay in a workgroup's registers, and longer ones."""
    a = head.inputs(R, V, C, seed=9, weights=True)
    ref = head.Exact(*a)
    head.agree(head.Call(rt, *a), ref)
    head.agree(head.Call(rt, *a, dx=False, dW=False), ref)


def test_many_rows_where_w_changes_size(rt):
    """64 tokens after the other whose largest values are far apart: each has a scale of its own, past 64 of them too."""
    x, W, t, w = head.inputs(MANY, 5000, 40, weights=True)
    rng = np.random.default_rng(13)
    W = (W * np.ldexp(1.0, rng.integers(-30, 1, (79, 1))).repeat(64, 0)[:5000]).astype(np.float32)
    W[128:192] = 0
    W[192:256] = 1e-38
    a = x, W, t, w
    head.agree(head.Call(rt, *a), head.Exact(*a))


@pytest.mark.parametrize("R,V,C", [(384, 50257, 20), (385, 50257, 20), (768, 50257, 20), (769, 50257, 20),
                                   (1152, 700, 400), (1153, 700, 400), (4096, 300, 50), (3000, 2000, 30)])
def test_where_w_is_laid_out_by_room(rt, R, V, C):
    a = head.inputs(R, V, C, seed=10, weights=True)
    ref = head.Exact(*a)
    head.agree(head.Call(rt, *a), ref)
    head.agree(head.Call(rt, *a, dx=False, dW=False), ref)
