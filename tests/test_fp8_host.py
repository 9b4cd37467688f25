"""8-bit floating point and clipping without a GPU: what the calls refuse before they touch a device."""
import pytest
import torch


def test_the_extension_refuses_tensors_that_are_not_on_the_device():
    from lancelot_b200._lib import InvalidArgument
    from lancelot_b200.pybind import _updates8 as m

    v, codes, scales = torch.zeros(2, 64), torch.zeros(2, 64, dtype=torch.float8_e4m3fn), torch.zeros(2, 1)
    for call in (lambda: m.quantize_fp8(0, 0, v, 1, 5, None, None, None, None),
                 lambda: m.dequantize_fp8(0, 0, codes, scales, 1, None),
                 lambda: m.fp8_matmul(0, 0, codes, scales, codes, scales, 3, None),
                 lambda: m.clip_updates(0, 0, v, 1.0, None),
                 lambda: m.clip_updates(0, 0, [[v]], None, None)):
        with pytest.raises(InvalidArgument, match="cuda:0"):
            call()
    for call in (lambda: m.clip_updates(0, 0, [v], None, None), lambda: m.clip_updates(0, 0, [[3]], None, None), lambda: m.clip_updates(0, 0, 3, None, None)):
        with pytest.raises(InvalidArgument, match="list of tensors"):
            call()
    with pytest.raises(InvalidArgument, match="not negative"):
        m.clip_updates(0, 0, [], -1.0, None)


class Made:
    """a sequence that makes its items when they are asked for, and keeps none"""

    def __init__(self, make, n, log=None, name=None):
        self.make, self.n, self.log, self.name = make, n, log if log is not None else [], name

    def __len__(self):
        return self.n

    def __getitem__(self, i):
        if i >= self.n:
            raise IndexError(i)
        self.log.append(("read", self.name))
        return self.make(i)

    def __del__(self):
        self.log.append(("gone", self.name))


def test_clients_that_are_made_on_access_are_held_while_they_are_read():
    from lancelot_b200._lib import InvalidArgument
    from lancelot_b200.pybind import _updates8 as m

    for out, most in ((None, None), (None, 1.0), (torch.zeros(2, 6), 1.0)):
        log = []
        updates = Made(lambda c: Made(lambda i: torch.zeros(3), 2, log, c), 2)
        with pytest.raises(InvalidArgument, match="cuda:0"):
            m.clip_updates(0, 0, updates, most, out)
        for c in range(2):
            mine = [what for what, name in log if name == c]
            assert mine and "gone" not in mine[:-1] and mine.count("read") == 2
    # an inner list that its owner fills anew for every client, and a sequence that fails
    box = []

    def refill(c):
        box[:] = [torch.zeros(3)]
        return box

    with pytest.raises(InvalidArgument, match="cuda:0"):
        m.clip_updates(0, 0, Made(refill, 3), 1.0, None)
    with pytest.raises(ZeroDivisionError):
        m.clip_updates(0, 0, Made(lambda c: 1 // 0, 3), 1.0, None)
    with pytest.raises(ZeroDivisionError):
        m.clip_updates(0, 0, [Made(lambda c: 1 // 0, 3)], 1.0, None)


def operand(codes, stride, across=0, code_type=5, scales=4096, scale_row=1, scale_block=1, scale_rows=1):
    import ctypes as C

    class S(C.Structure):
        _fields_ = [("codes", C.c_void_p), ("stride", C.c_int64), ("across", C.c_int), ("code_type", C.c_int), ("scales", C.c_void_p), ("scale_row", C.c_int64),
                    ("scale_block", C.c_int64), ("scale_rows", C.c_int)]

    return S(codes, stride, across, code_type, scales, scale_row, scale_block, scale_rows)


def test_the_c_entries_refuse_a_null_context():
    import ctypes as C

    from lancelot_b200 import lib

    z, n, f = C.c_int64(0), None, C.c_size_t(0)
    assert lib.lb_quantize_fp8(n, n, 1, z, z, z, 1, 5, n, z, n, z, n, z, n, z, n) == 1
    assert lib.lb_dequantize_fp8(n, n, 5, z, n, z, 1, z, z, n, 1, z, n) == 1
    assert lib.lb_fp8_matmul(n, z, z, z, n, n, n, 1, z, n, f, n) == 1
    assert lib.lb_clip_updates(n, 0, 0, n, n, n, n, C.c_double(1), n, n, n, n, f, n) == 1
    assert b"context" in lib.lb_last_error()


def test_a_product_asks_for_a_workspace_only_where_rows_are_off_their_alignment():
    import ctypes as C

    from lancelot_b200 import lib

    f = lib.lb_fp8_matmul_workspace_bytes
    f.restype = C.c_size_t
    i = C.c_int64
    need = lambda m, n, k, a, b: f(i(m), i(n), i(k), C.byref(a), C.byref(b))  # noqa: E731
    fine = operand(1 << 20, 256)
    assert need(300, 500, 200, fine, fine) == 0 and need(0, 5, 200, fine, fine) == 0 and f(i(5), i(5), i(5), None, None) == 0
    assert need(300, 500, 200, operand((1 << 20) + 1, 256), fine) == -(-300 * 208 // 256) * 256
    assert need(300, 500, 200, operand(1 << 20, 333, across=1), operand(1 << 20, 200)) == -(-200 * 304 // 256) * 256 + -(-500 * 208 // 256) * 256


def test_clipping_asks_for_a_sum_for_every_piece():
    import ctypes as C

    from lancelot_b200 import lib

    f = lib.lb_clip_updates_workspace_bytes
    f.restype = C.c_size_t
    sizes = (C.c_int64 * 4)(1, 1024, 1025, 0)
    assert f(2, 4, sizes) == 8 * (2 + 1 + 1 + 2) and f(3, 0, None) == 24
    assert f(0, 4, sizes) == 0 and f(2, 4, None) == 0 and f(1, 1, (C.c_int64 * 1)(-5)) == 0


def test_a_layer_checks_its_shapes():
    from lancelot_b200 import updates

    for x, w in (((3, 4), (5, 3)), ((3, 4), (4,)), ((), (4, 4))):
        with pytest.raises(ValueError):
            updates.fp8_linear(None, torch.zeros(x), torch.zeros(w))
    with pytest.raises(ValueError):
        updates.fp8_linear(None, torch.zeros(3, 4), torch.zeros(5, 4), grad_dtype=torch.float32)
    with pytest.raises(ValueError, match="different numbers"):
        updates.flat_updates(None, [[torch.zeros(3)], [torch.zeros(4)]])
