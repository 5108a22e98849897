"""Whether tensors share memory (dgen_hip._tensor_args.covers) against the sets
of their bytes."""
import itertools

import pytest

torch = pytest.importorskip("torch")

from dgen_hip._tensor_args import covers  # noqa: E402


def bytes_of(t):
    at = [t.data_ptr() + t.itemsize * sum(i * s for i, s in zip(index, t.stride()))
          for index in itertools.product(*(range(n) for n in t.shape))]
    return {a + k for a in at for k in range(t.itemsize)}


def views(t):
    """Of a float32 tensor [4][6][10]."""
    half = t.view(torch.bfloat16)  # [4][6][20]
    return [t, t[..., :5], t[..., 5:], t[..., 4:6], t[:2], t[2:], t[:, :3], t[:, 3:], t[:, 1::2], t[:, ::2], t[:1],
            t[3:], t[:, :, ::2], t.transpose(0, 1), t.transpose(1, 2), t[1:2].expand(4, 6, 10),
            t[..., :1].expand(4, 6, 10), t[:0], t[0], t[:, 0], t[0, 0], t[0, 0, 0], t[1:3, 2:5, 3:7], t.view(24, 10),
            t.view(24, 10)[1:], t.view(240)[3:11], t.view(240).as_strided((5, 7), (20, 1), 13),
            t.view(240).as_strided((5, 7), (9, 1), 4), half, half[..., :10], half[..., 10:], half[..., 9:11],
            half[:, 2]]


def test_against_the_sets_of_bytes():
    t = torch.zeros(4, 6, 10)
    all_views = views(t) + [torch.zeros(4, 6, 10)]
    held = [bytes_of(v) for v in all_views]
    apart = told = 0
    for (a, x), (b, y) in itertools.product(zip(all_views, held), repeat=2):
        got, exact = covers(0, a, b), covers(1, a, b)
        if x & y:
            assert got is True, (a.shape, a.stride(), b.shape, b.stride())
            same = a.data_ptr() == b.data_ptr() and a.dtype == b.dtype and a.shape == b.shape and all(
                n == 1 or p == q for n, p, q in zip(a.shape, a.stride(), b.stride()))
            assert exact is (not same)
        else:
            apart += 1
            told += not got
            assert exact is got
    # (which columns, rows or sequences are taken side by side is told; a few interleaved layouts are not)
    assert told >= 0.9 * apart, (told, apart)
    for a, b in ((t[..., :5], t[..., 5:]), (t[:2], t[2:]), (t[:, :3], t[:, 3:]), (t[:, 0], t[:, 1]),
                 (t[:, :3, :5], t[:, 2:, 5:]), (t[:, ::2], t[:, 1::2])):
        assert covers(0, a, b) is False and covers(0, b, a) is False


def test_the_first_may_be_the_tensor_itself():
    t = torch.zeros(3, 8)
    assert covers(0, t, t) is True and covers(1, t, t) is False and covers(1, t, None, t) is True
    assert covers(2, t, None, t) is False and covers(1, t, t, torch.zeros(2), None) is False
    assert covers(1, t, t, t[1]) is True and covers(9, t, t[1:]) is True
    assert covers(0, t, None) is False and covers(0, t) is False and covers(0, t[:0], t) is False
    for wrong in ((), (0,), (0, "t"), (0, t, "t"), ("a", t, t)):
        assert covers(*wrong) is None
