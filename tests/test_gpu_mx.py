"""GPU: MXFP4 tables (lgx_mx_quantize / lgx_mx_dequantize) and the scores over them (lgx_score_mx).

The packed form is a definition without rounding freedom, so quantisation is compared bit by bit with its
definition in 64 bits.  Scores: the products of two decoded elements are exact in f32, so only the sum of
d of them rounds; with every addition off by at most one step (2^-23 of the partial sum, whatever the
rounding direction of the matrix instruction) |error| <= d 2^-23 sum_k |q_k t_k|."""
import numpy as np
import pytest
import torch

import factors_of_serendipity_recommendation_amd as lgx
from factors_of_serendipity_recommendation_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
LEVELS = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def ref_pack(x):
    """(codes [rows, 32 nb], scale bytes [rows, nb]) of float64 rows, from the definition."""
    rows, d = x.shape
    nb = -(-d // 32)
    b = np.zeros((rows, nb * 32))
    b[:, :d] = x
    b = b.reshape(rows, nb, 32)
    a = np.abs(b).max(2)
    bad = ~np.isfinite(b).all(2)
    with np.errstate(all="ignore"):
        e = np.where(a > 0, np.frexp(np.where(bad, 1.0, a))[1] - 1, -1000)
    byte = np.where(bad, 255, np.clip(e - 2, -127, 127) + 127)
    y = np.abs(np.where(bad[..., None], 0.0, b)) * 2.0 ** (127.0 - np.where(bad, 127, byte))[..., None]
    dist = np.abs(np.minimum(y, 6.0)[..., None] - LEVELS)
    best = dist.min(-1, keepdims=True)
    order = [0, 2, 4, 6, 1, 3, 5, 7]  # an even code wins a tie
    pick = np.array(order)[(dist == best)[..., order].argmax(-1)]
    code = np.where(bad[..., None], 0, pick + 8 * np.signbit(b))
    return code.reshape(rows, nb * 32).astype(np.uint8), byte.astype(np.uint8)


def ref_values(codes, scales, d):
    v = np.where(codes & 8, -1.0, 1.0) * LEVELS[codes & 7]
    s = np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.float64) - 127))
    return (v.reshape(*scales.shape, 32) * s[..., None]).reshape(codes.shape)[:, :d]


def nibbles(t):
    c = t.codes.cpu().numpy()
    return np.stack((c & 15, c >> 4), 2).reshape(c.shape[0], 2 * c.shape[1])


def table(rows, d, seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, d, generator=g) * torch.exp(torch.randn(rows, 1, generator=g))
    return x.to(dtype).to(DEV)


def values64(t):
    return torch.from_numpy(ref_values(nibbles(t), t.scales.cpu().numpy(), t.d))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,d", [(1, 1), (3, 31), (5, 32), (7, 33), (1000, 64), (129, 100), (65, 256), (2, 1000),
                                    (1, 4099), (257, 40)])
def test_quantize_matches_its_definition(rows, d, dtype):
    x = table(rows, d, rows * 131 + d, dtype)
    t = lgx.mx_quantize(x)
    codes, scales = ref_pack(x.double().cpu().numpy())
    assert t.shape == (rows, d) and np.array_equal(t.scales.cpu().numpy(), scales)
    assert np.array_equal(nibbles(t), codes)
    want = torch.from_numpy(ref_values(codes, scales, d))
    for out in (torch.float32, torch.bfloat16):
        got = lgx.mx_dequantize(t, out)
        assert got.dtype == out and torch.equal(got.double().cpu(), want)


def test_quantize_borders_extremes_and_non_finite_blocks():
    """Every border between two magnitudes (ties to the even code) and the f32 steps beside it, both signs,
    at scales from the largest to subnormal ones; zero blocks; blocks with an infinity or a NaN."""
    border = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=np.float32)
    v = np.concatenate([border, np.nextafter(border, np.float32(0)), np.nextafter(border, np.float32(9)),
                        [4, 6, np.nextafter(np.float32(8), np.float32(0)), 0, -0.0]]).astype(np.float32)
    block = np.zeros(32, np.float32)
    block[:26] = v
    rows = [block * np.float32(s) * np.float32(2.0 ** e) for s in (1, -1) for e in (0, 100, 125, -60, -120, -124)]
    rows += [np.zeros(32, np.float32), np.full(32, 1e-45, np.float32), np.full(32, 2.0 ** -126, np.float32),
             np.full(32, np.finfo(np.float32).max), np.full(32, -6 * 2.0 ** -129, np.float32)]
    for bad in (np.inf, -np.inf, np.nan):
        r = block.copy()
        r[31] = bad
        rows.append(r)
    x = np.stack(rows)
    x = np.concatenate([x, np.roll(x, 1, 0)], 1)  # a bad block leaves its neighbour alone
    t = lgx.mx_quantize(torch.from_numpy(x).to(DEV))
    codes, scales = ref_pack(x.astype(np.float64))
    assert np.array_equal(t.scales.cpu().numpy(), scales) and np.array_equal(nibbles(t), codes)
    want = ref_values(codes, scales, 64)
    for out in (torch.float32, torch.bfloat16):
        got = lgx.mx_dequantize(t, out).double().cpu().numpy()
        assert np.array_equal(got, want, equal_nan=True)
    assert np.isnan(want[-3:, :32]).all() and not np.isnan(want[1]).any()


def test_quantize_takes_strided_rows_and_no_rows():
    base = table(50, 200, 5)
    for x in (base[:, 8:108], base[:, 3:67], base[::3, :64], base.t(), base[:1].expand(4, 200), base[:0], base[5:6, 1:]):
        t = lgx.mx_quantize(x)
        codes, scales = ref_pack(x.double().cpu().numpy())
        assert t.shape == tuple(x.shape)
        assert np.array_equal(nibbles(t), codes) and np.array_equal(t.scales.cpu().numpy(), scales)
        assert lgx.mx_dequantize(t).shape == x.shape


def score_bound(q, it):
    return q.shape[1] * 2.0 ** -23 * (q.abs() @ it.abs().T) + 1e-30


@pytest.mark.parametrize("B,I,d", [(1, 1, 1), (1, 1000, 64), (2, 129, 32), (31, 513, 33), (33, 511, 256), (70, 2120, 100),
                                   (130, 700, 290), (5, 4097, 320), (64, 300, 1000), (257, 640, 64), (40, 1025, 160),
                                   (300, 130, 512)])
@pytest.mark.parametrize("kind", ["f32", "bf16", "mx"])
def test_score_mx_matches_64_bits(B, I, d, kind):
    x = table(B, d, B + I + d, torch.bfloat16 if kind == "bf16" else torch.float32)
    items = lgx.mx_quantize(table(I, d, I))
    packed = lgx.mx_quantize(x)
    q, it = values64(packed), values64(items)
    want, bound = q @ it.T, score_bound(q, it)
    arg = packed if kind == "mx" else x
    got = lgx.score_mx(arg, items).double().cpu()
    assert ((got - want).abs() <= bound).all()
    got = lgx.score_mx(arg, items, dtype=torch.bfloat16)
    assert got.dtype == torch.bfloat16
    assert ((got.double().cpu() - want).abs() <= bound + 2.0 ** -8 * (want.abs() + bound)).all()
    # sigmoid: a slope of at most 1/4 of the score's error, exp within 2^-21 relative, one addition and
    # one division
    got = lgx.score_mx(arg, items, apply_sigmoid=True).double().cpu()
    assert ((got - torch.sigmoid(want)).abs() <= bound / 4 + 2.0 ** -20).all()


@pytest.mark.parametrize("B,I,d,scale", [(5, 700, 64, 0.5), (70, 641, 100, 1.0), (40, 300, 600, 0.5), (300, 1000, 64, 8.0)])
def test_sigmoid_in_bf16(B, I, d, scale):
    """One rounding to bf16 beside the score's own error (a slope of at most 1/4) and the f32 arithmetic's; scores of hundreds
    end at 0 and 1."""
    t, items = lgx.mx_quantize(table(B, d, B) * scale), lgx.mx_quantize(table(I, d, I) * scale)
    q, it = values64(t), values64(items)
    want, bound = torch.sigmoid(q @ it.T), score_bound(q, it)
    got = lgx.score_mx(t, items, apply_sigmoid=True, dtype=torch.bfloat16).double().cpu()
    assert ((got - want).abs() <= bound / 4 + 2.0 ** -17 * want + 2.0 ** -9 * (want + bound) * 2 + 1e-38).all()


@pytest.mark.parametrize("B,d", [(3, 64), (50, 100), (50, 300)])
def test_sigmoid_of_infinite_and_undefined_scores(B, d):
    """Scores past f32's range are 0 and 1, undefined ones stay so."""
    x, y = torch.full((B, d), 1e30, device=DEV), torch.full((7, d), 1e30, device=DEV)
    y[1], y[2], y[3, 0], y[4] = -1e30, 0.0, float("nan"), 1e-30
    q, it = lgx.mx_quantize(x), lgx.mx_quantize(y)
    raw = lgx.score_mx(q, it)
    assert (raw[:, 0] == float("inf")).all() and (raw[:, 1] == float("-inf")).all()
    want = torch.tensor([1.0, 0.0, 0.5, float("nan"), 1.0, 1.0, 1.0], device=DEV).expand(B, 7)
    for dtype in (torch.float32, torch.bfloat16):
        got = lgx.score_mx(q, it, apply_sigmoid=True, dtype=dtype).float()
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(torch.nan_to_num(got, 7.0), torch.nan_to_num(want, 7.0))


@pytest.mark.parametrize("kind", ["f32", "mx"])
def test_score_mx_gathers_rows_and_flags_bad_ones(kind):
    x, items = table(40, 96, 1), lgx.mx_quantize(table(333, 96, 2))
    q = lgx.mx_quantize(x)
    rows = torch.tensor([3, 3, 39, 0, -1, 40, 7, 2 ** 40, -2 ** 40], device=DEV)
    got = lgx.score_mx(q if kind == "mx" else x, items, user_rows=rows)
    ok = [0, 1, 2, 3, 6]
    want = lgx.score_mx(q, items)
    assert torch.equal(got[ok], want[rows[ok]])
    assert torch.isnan(got[[4, 5, 7, 8]]).all()
    assert lgx.score_mx(q, items, user_rows=rows[:0]).shape == (0, 333)
    assert lgx.score_mx(q, items[:0]).shape == (40, 0)
    assert torch.equal(lgx.score_mx(q[3:9], items[100:200]), want[3:9, 100:200])


@pytest.mark.parametrize("kind", ["f32", "bf16", "mx"])
@pytest.mark.parametrize("B,d", [(20, 90), (32, 256), (50, 64), (40, 600), (100, 290)])
def test_rows_outside_the_table_and_undefined_blocks_of_every_form(B, d, kind):
    """Strided queries at odd addresses, repeated and outside rows, NaN blocks at both ends of a row: each reaches its own
    scores only, and in every form of the product the rest equals the same rows scored one by one."""
    base = table(64, d + 9, B, torch.bfloat16 if kind == "bf16" else torch.float32)
    base[2, 3 + d - 1], base[5, 3] = float("inf"), float("nan")
    x, y = base[:, 3:3 + d], table(777, d, d)
    y[4, 0], y[700, d - 1] = float("nan"), float("-inf")
    items = lgx.mx_quantize(y)
    rows = torch.randint(0, 64, (B,), generator=torch.Generator().manual_seed(d)).to(DEV)
    rows[1], rows[7], rows[B - 1], rows[B - 2], rows[3] = -1, 64, 2 ** 33, 5, 2
    got = lgx.score_mx(lgx.mx_quantize(x) if kind == "mx" else x, items, user_rows=rows)
    outside = (rows < 0) | (rows >= 64)
    bad = (outside | (rows == 2) | (rows == 5))[:, None].expand(B, 777).clone()
    bad[:, 4], bad[:, 700] = True, True
    assert torch.equal(torch.isnan(got), bad)
    for j in (0, 2, B // 2, B - 3):
        if not bad[j, 0]:
            one = lgx.score_mx(lgx.mx_quantize(x), items, user_rows=rows[j:j + 1])
            assert torch.equal(torch.nan_to_num(got[j], 7.0), torch.nan_to_num(one[0], 7.0))


def test_rows_of_an_empty_table():
    """Every row lies outside it."""
    for B, d in ((3, 64), (50, 64), (3, 320), (50, 320)):
        x, it = torch.empty(0, d, device=DEV), lgx.mx_quantize(table(100, d, 1))
        rows = torch.arange(B, device=DEV)
        for q in (x, x.bfloat16(), lgx.mx_quantize(x)):
            assert torch.isnan(lgx.score_mx(q, it, user_rows=rows)).all()
            assert lgx.score_mx(q, it).shape == (0, 100)


def test_score_mx_keeps_a_nan_block_to_its_rows():
    x, y = table(4, 64, 1), table(200, 64, 2)
    x[1, 5], y[17, 60] = float("nan"), float("inf")
    got = lgx.score_mx(x, lgx.mx_quantize(y))
    bad = torch.zeros(4, 200, dtype=torch.bool, device=DEV)
    bad[1], bad[:, 17] = True, True
    assert torch.equal(torch.isnan(got), bad)


def test_score_mx_spans_the_scale_range():
    """Scales from 2^-60 to 2^60 in one row's blocks: the products keep their own exponents."""
    g = torch.Generator().manual_seed(3)
    e = torch.randint(-60, 60, (20, 8, 1), generator=g).double()
    x = (torch.randn(20, 8, 32, generator=g).double() * 2.0 ** e).view(20, 256).float().to(DEV)
    y = (torch.randn(150, 8, 32, generator=g).double() * 2.0 ** torch.randint(-60, 60, (150, 8, 1), generator=g)).view(150, 256)
    t, it = lgx.mx_quantize(x), lgx.mx_quantize(y.float().to(DEV))
    q, v = values64(t), values64(it)
    assert ((lgx.score_mx(t, it).double().cpu() - q @ v.T).abs() <= score_bound(q, v)).all()


def test_score_mx_into_out_leaves_the_rest_alone():
    t, it = lgx.mx_quantize(table(37, 64, 1)), lgx.mx_quantize(table(1001, 64, 2))
    buf = torch.full((40, 1001), 7.0, device=DEV)
    out = lgx.score_mx(t, it, out=buf[1:38])
    assert out.data_ptr() == buf[1:].data_ptr()
    assert torch.equal(buf[1:38], lgx.score_mx(t, it))
    assert (buf[0] == 7).all() and (buf[38:] == 7).all()


def test_tables_pass_2_31_bytes_of_scores():
    """A score matrix past 2^31 elements: the last rows and columns are the ones of the small call."""
    t, it = lgx.mx_quantize(table(2200, 32, 1)), lgx.mx_quantize(table(1000000, 32, 2))
    S = lgx.score_mx(t, it, dtype=torch.bfloat16)
    want = lgx.score_mx(t[2190:], it[999000:], dtype=torch.bfloat16)
    assert torch.equal(S[2190:, 999000:], want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_more_rows_than_a_launch_takes(dtype):
    """2^30 rows of one element: four launches' blocks, of more threads than one grid holds.  A row of one element x is
    +-4 scales, where x lies below 5 of them, or 6."""
    rows, part = 2 ** 30 + 3, 2 ** 27
    x = torch.empty(rows, 1, dtype=dtype, device=DEV)
    for r in x.split(part):
        r.normal_()
    t = lgx.mx_quantize(x)
    back = lgx.mx_dequantize(t, torch.bfloat16)
    for a in range(0, rows, part):
        v = x[a:a + part].float()
        unit = torch.exp2(torch.floor(torch.log2(v.abs().double()).clamp(min=-140)) - 2).float()
        unit = torch.where(v.abs() >= 8 * unit, unit * 2, torch.where(v.abs() < 4 * unit, unit / 2, unit))  # log2 rounds
        want = torch.where(v.abs() <= 5 * unit, 4 * unit, 6 * unit) * torch.sign(v)
        assert torch.equal(back[a:a + part].float(), want)
        del v, unit, want


@pytest.mark.parametrize("B,d,kind", [(2 ** 24 + 300, 40, "f32"), (2 ** 24 + 300, 40, "mx"), (2 ** 22 + 1, 64, "f32"),
                                      (2 ** 22 + 1, 64, "mx"), (2 ** 22 + 1, 290, "f32"), (2 ** 28 + 129, 290, "mx")])
def test_more_queries_than_a_launch_takes(B, d, kind):
    """Millions of queries of a few rows: each scores what the row scores in a small batch."""
    x, items = table(7, d, d), lgx.mx_quantize(table(1 if B > 2 ** 27 else 3, d, 2))
    q = lgx.mx_quantize(x) if kind == "mx" else x
    few = torch.arange(50, device=DEV) % 7
    want = lgx.score_mx(q, items, user_rows=few)[:7]
    rows = torch.randint(0, 7, (B,), device=DEV, generator=torch.Generator(device=DEV).manual_seed(d))
    rows[-1], rows[-2] = 7, 3  # outside: NaN
    got = lgx.score_mx(q, items, user_rows=rows)
    assert torch.isnan(got[-1]).all()
    assert torch.equal(got[:-1], want[rows[:-1]])
    if kind == "mx" and B < 2 ** 23:  # and rows without a list
        many = lgx.MXTable(q.codes[rows % 7], q.scales[rows % 7], d)
        assert torch.equal(lgx.score_mx(many, items), want[rows % 7])


def test_mx_refusals():
    x = table(4, 64, 1)
    t = lgx.mx_quantize(x)
    with pytest.raises(TypeError):
        lgx.mx_quantize(x.half())
    with pytest.raises(ValueError):
        lgx.mx_quantize(x[0])
    with pytest.raises(RuntimeError, match="65537"):
        lgx.mx_quantize(torch.zeros(1, 65537, device=DEV))
    with pytest.raises(TypeError):
        lgx.mx_dequantize(t, torch.float16)
    with pytest.raises(TypeError):
        lgx.score_mx(x, x)
    with pytest.raises(ValueError):
        lgx.score_mx(x[:, :32], t)
    with pytest.raises(TypeError):
        lgx.score_mx(x, t, dtype=torch.float16)
    with pytest.raises(ValueError):
        lgx.score_mx(x, t, out=torch.empty(4, 5, device=DEV))
    with pytest.raises(ValueError):
        lgx.score_mx(x, t.to("cpu").to(DEV), user_rows=torch.zeros(2, 2, dtype=torch.long, device=DEV))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        lgx.score_mx(x.cpu(), t)


def test_model_scores_against_a_quantised_catalog(mlls):
    """LightGCN.getUsersRating over quantizeItems(): the scores of the propagated tables' packed rows."""
    class _DS:
        pass

    ds = _DS()
    ds.n_users, ds.m_items = int(mlls["n_users"]), int(mlls["n_items"])
    A = lgx.build_norm_adj(mlls["train_users"], mlls["train_items"], ds.n_users, ds.m_items, dedup=True, device=DEV)
    ds.getSparseGraph = lambda: None
    ds.getCSRGraph = lambda: A
    from factors_of_serendipity_recommendation_amd.model import LightGCN
    torch.manual_seed(3)
    model = LightGCN({"latent_dim_rec": 64, "lightGCN_n_layers": 3, "pretrain": 0, "dropout": 0}, ds).to(DEV).eval()
    users = torch.tensor([5, 0, ds.n_users - 1], device=DEV)
    with torch.no_grad():
        eu, ei = model.computer()
        items = model.quantizeItems()
        got = model.getUsersRating(users, items)
    assert torch.equal(items.codes, lgx.mx_quantize(ei).codes)
    assert torch.equal(got, ops.score_mx(eu[users], items, apply_sigmoid=True))
