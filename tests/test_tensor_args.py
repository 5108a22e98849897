"""The native tests of tensor arguments against the ones in Python, which say
what is wrong with an argument."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from dgen_hip import sequence as Q  # noqa: E402
from dgen_hip._tensor_args import dense, rows, sequence  # noqa: E402

F32, BF16, INT32 = 0, 1, 2


def test_what_is_no_device_tensor_is_turned_down():
    x = torch.zeros(2, 3, 4)
    for f in (dense, rows, sequence):
        for index in (-1, 0):
            assert f(x, x.shape, F32, index) is None  # on the host
        assert f("x", (2, 3, 4), F32, 0) is None
        assert f(x, [2, 3, 4], F32, 0) is None
        assert f(x, ("a", 3, 4), F32, 0) is None
        assert f(x, x.shape, "a", 0) is None
        assert f(x, x.shape, 7, 0) is None
        assert f(x) is None
        assert f() is None
        assert f(x.to_sparse(), x.shape, F32, 0) is None
        assert f(torch.empty(2, 3, 4, device="meta"), x.shape, F32, 0) is None
    assert dense(None, (4,), F32, 0) == 0 and rows(None, (4,), F32, 0) is None and sequence(None, (4,), F32, 0) is None


def views():
    for dtype, code in ((torch.float32, F32), (torch.bfloat16, BF16), (torch.int32, INT32)):
        t = torch.zeros(6, 10, 16, dtype=dtype, device="cuda")
        for v in (t, t[1:, 2:5, 3:], t[:, :, :1], t[:, :, ::2], t.transpose(0, 1), t.transpose(1, 2), t[:0], t[0], t[:, 3],
                  t[0, 0], t[1:2].expand(6, 10, 16), t[..., :1].expand(6, 10, 16), t.new_zeros(()), t.new_zeros(4, 1).t(),
                  torch.nn.Parameter(t[:2], requires_grad=False)):
            yield v, code


@pytest.mark.gpu
def test_the_same_as_in_python():
    def tried(f, *args):
        try:
            return f(*args)
        except ValueError:
            return None

    seen = 0
    for v, code in views():
        for shape in (v.shape, (*v.shape, 1), (7, *v.shape[1:])):
            for dtype, c in ((torch.float32, F32), (torch.bfloat16, BF16), (torch.int32, INT32)):
                args = v, "v", shape, dtype, torch.device("cuda", 0)
                got = dense(v, shape, c, 0)
                assert got == tried(Q._dense, *args)
                if len(shape) == 3:
                    assert sequence(v, shape, c, 0) == tried(Q._seq, *args)
                if len(shape) >= 1 and len(shape) == v.dim():
                    got, want = rows(v, shape, c, 0), tried(Q._rows, *args)
                    # (folding the leading axes of a view is left to the one in Python)
                    assert got == want or (got is None and want is not None and v.dim() != 2)
                seen += got is not None
        assert dense(v, v.shape, code, 1) is None
    assert seen > 20
