"""CPU: argument checks of the MXFP4 and sampling entry points (no device work)."""
import ctypes

import pytest
import torch

import factors_of_serendipity_recommendation_amd as lgx
from factors_of_serendipity_recommendation_amd import _lib, ops, recommend

P = ctypes.c_void_p(4096)  # an aligned address that a refused call never touches
ODD = ctypes.c_void_p(4100)


def _err():
    return _lib.lib().lgx_last_error()


def test_mxtable_checks_its_parts():
    c, s = torch.zeros(3, 32, dtype=torch.uint8), torch.zeros(3, 2, dtype=torch.uint8)
    t = lgx.MXTable(c, s, 40)
    assert t.shape == (3, 40) and len(t) == 3 and t[1:].shape == (2, 40) and len(t[:0]) == 0
    assert t.to("cpu").codes.shape == c.shape
    for bad in ((c, s, 65), (c, s, 0), (c[:2], s, 40), (c[:, :16], s, 40), (c, s[:, :1], 40), (c[0], s, 40)):
        with pytest.raises(ValueError):
            lgx.MXTable(*bad)
    with pytest.raises(TypeError):
        lgx.MXTable(c.int(), s, 40)
    with pytest.raises(ValueError):
        lgx.MXTable(torch.zeros(3, 64, dtype=torch.uint8)[:, ::2], s, 40)
    with pytest.raises(ValueError):
        lgx.MXTable(torch.zeros(97, dtype=torch.uint8)[1:].view(3, 32), s, 40)
    with pytest.raises(TypeError):
        t[1]
    with pytest.raises(TypeError):
        t[::2]


def test_new_ops_refuse_cpu_tensors():
    x = torch.zeros(4, 64)
    t = lgx.MXTable(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8), 64)
    for call in (lambda: lgx.mx_quantize(x), lambda: lgx.mx_dequantize(t), lambda: lgx.score_mx(x, t),
                 lambda: lgx.score_mx(t, t), lambda: lgx.sample_rows(x, torch.zeros(4))):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


def test_quantize_entry_points_refuse_bad_arguments():
    L = _lib.lib()
    assert L.lgx_mx_quantize(None, 0, 64, 64, 0, None, None, None) == 0       # no rows: nothing to do
    assert L.lgx_mx_quantize(None, 1, 64, 64, 0, P, P, None) == 1
    assert L.lgx_mx_quantize(P, -1, 64, 64, 0, P, P, None) == 1
    assert L.lgx_mx_quantize(P, 1, 64, 64, 2, P, P, None) == 1                # a packed source
    assert L.lgx_mx_quantize(P, 1, 0, 64, 0, P, P, None) == 3
    assert L.lgx_mx_quantize(P, 1, 65537, 65537, 0, P, P, None) == 3
    assert L.lgx_mx_quantize(P, 2, 64, 63, 0, P, P, None) == 3 and b"ld=63" in _err()
    assert L.lgx_mx_quantize(P, 1, 64, 64, 0, ODD, P, None) == 1 and b"16-byte" in _err()
    assert L.lgx_mx_quantize(P, 2 ** 40, 64, 64, 0, P, P, None) == 3
    assert L.lgx_mx_dequantize(P, P, 1, 64, 7, P, None) == 1
    assert L.lgx_mx_dequantize(P, None, 1, 64, 0, P, None) == 1
    assert L.lgx_mx_dequantize(P, P, 1, 0, 0, P, None) == 3
    assert L.lgx_mx_dequantize(ODD, P, 1, 64, 0, P, None) == 1


def test_score_entry_point_refuses_bad_arguments():
    L = _lib.lib()
    ws = ctypes.c_size_t()
    assert L.lgx_score_mx_workspace(10, 100, 2, ctypes.byref(ws)) == 0 and ws.value == 0
    assert L.lgx_score_mx_workspace(40, 100, 0, ctypes.byref(ws)) == 0 and ws.value >= 40 * 4 * 17
    assert L.lgx_score_mx_workspace(10, 0, 0, ctypes.byref(ws)) == 1

    def call(Q=P, qs=P, qd=2, n_q=40, ld=0, rows=None, codes=P, scales=P, B=40, n=100, d=64, od=0, out=P, work=None, wb=0):
        return L.lgx_score_mx(Q, qs, qd, n_q, ld, rows, codes, scales, B, n, d, 0, od, out, work, wb, None)

    assert call(B=0) == 0 and call(n=0) == 0
    assert call(B=-1) == 1 and call(n=-1) == 1
    assert call(qd=3) == 1 and call(od=2) == 1
    assert call(d=0) == 3 and call(d=65537) == 3
    assert call(n=2 ** 31) == 3
    assert call(Q=None) == 1 and call(codes=None) == 1 and call(scales=None) == 1 and call(out=None) == 1
    assert call(B=41) == 1 and b"41 queries of 40 rows" in _err()
    assert call(codes=ODD) == 1 and call(Q=ODD) == 1 and call(qs=None) == 1
    assert call(qd=0, ld=63, work=P, wb=1 << 20) == 1
    assert call(qd=0, ld=64) == 4 and b"workspace" in _err()
    assert call(qd=0, ld=64, work=P, wb=16) == 4


def test_sample_entry_point_refuses_bad_arguments():
    L = _lib.lib()
    ws = ctypes.c_size_t()
    assert L.lgx_sample_rows_workspace(4, 100, 1, ctypes.byref(ws)) == 0
    assert L.lgx_sample_rows_workspace(4, 0, 1, ctypes.byref(ws)) == 1

    def call(S=P, dt=0, rows=4, cols=100, ld=100, u=P, ud=0, n=1, idx=P):
        L.lgx_sample_rows_workspace(max(rows, 0), max(cols, 1), max(n, 0), ctypes.byref(ws))
        return L.lgx_sample_rows(S, dt, rows, cols, ld, u, ud, n, 1.0, None, 0, None, 1.0, None, 0.0, None, idx, None, P,
                                 ws.value, None)

    assert call(rows=0) == 0 and call(n=0) == 0
    assert call(rows=-1) == 1 and call(n=-1) == 1
    assert call(dt=2) == 1 and call(ud=1) == 1
    assert call(cols=0) == 1 and call(cols=2 ** 31, ld=2 ** 31) == 1 and call(ld=99) == 1
    assert call(rows=2 ** 31) == 3
    assert call(S=None) == 1 and call(u=None) == 1 and call(idx=None) == 1


def test_sample_entry_point_of_64_bit_settings_refuses_the_same():
    L = _lib.lib()

    def call(S=P, rows=4, cols=100, ld=100, u=P, ud=0, idx=P):
        return L.lgx_sample_rows_f64(S, 0, rows, cols, ld, u, ud, 1, 1.0, P, 0, None, 1.0, P, 0.0, P, idx, None, None, 0, None)

    assert call(rows=0) == 0
    assert call(rows=-1) == 1 and call(ud=1) == 1 and call(cols=0) == 1 and call(ld=99) == 1
    assert call(rows=2 ** 31) == 3
    assert call(S=None) == 1 and call(u=None) == 1 and call(idx=None) == 1
    assert call(rows=1, cols=100000, ld=100000) == 4 and b"workspace" in _err()


def test_mask_of_sample_recommendations_is_checked():
    ip, ix = torch.tensor([0, 2, 2, 3]), torch.tensor([0, 9, 4], dtype=torch.int32)
    check = recommend._check_mask
    check((ip, ix), 3, 10)
    check((torch.zeros(1, dtype=torch.int64), ix[:0]), 0, 10)
    check((torch.zeros(4, dtype=torch.int64), ix[:0]), 3, 0)
    for bad in ((ip, ix, 2, 10), (ip[:-1], ix, 2, 10), (ip + 1, ix, 3, 10), (torch.tensor([0, 3, 2, 3]), ix, 3, 10),
                (ip.view(2, 2), ix, 3, 10), (ip, ix.view(1, 3), 3, 10)):
        with pytest.raises(ValueError):
            check(bad[:2], *bad[2:])
    for indices, n_items in ((ix, 9), (ix - 1, 10)):
        with pytest.raises(IndexError):
            check((ip, indices), 3, n_items)
    for types in ((ip.int(), ix), (ip, ix.long()), (ip.float(), ix)):
        with pytest.raises(TypeError):
            check(types, 3, 10)


def test_mask_of_empty_lists():
    """What the framework itself makes of lists without an item: an indptr of zeros and a single index."""
    for users in (0, 1, 3):
        mask = ops.lists_to_device_csr([[] for _ in range(users)], "cpu")
        for n_items in (0, 1, 10):
            recommend._check_mask(mask, users, n_items)
        assert not ops.dense_mask_offsets(mask, 10, 0, users).numel()
    zeros = torch.zeros(3, dtype=torch.int64)
    with pytest.raises(ValueError):
        recommend._check_mask((zeros, torch.zeros(2, dtype=torch.int32)), 2, 10)
    with pytest.raises(ValueError):
        recommend._check_mask((torch.tensor([0, 1, 0]), torch.zeros(1, dtype=torch.int32)), 2, 10)
    with pytest.raises(ValueError):
        recommend._check_mask((zeros + 1, torch.zeros(1, dtype=torch.int32)), 2, 10)
