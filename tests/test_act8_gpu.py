"""Rows held in 8 bits (det3d_amd/act8.py, csrc/d3d_act8.hip) on the GPU: which values come back (against the definition in 64
bits, bit for bit), the weight gradient that reads the codes (against float64 sums), layouts, edges, streams and graphs."""
import pytest
import torch

pytestmark = pytest.mark.gpu

EPS32 = 2.0 ** -24  # half a step of float32, relative


@pytest.fixture(scope="module")
def act8(hip_lib):
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from det3d_amd import act8 as m

    return m


def power(s):
    return ((s.to(torch.int64) + 1023) << 52).view(torch.float64)


def restored(x, fmt):
    """the held values by definition, float64 on the CPU"""
    x = x.detach().cpu().double()
    n, c = x.shape
    v = torch.zeros(n, (c + 31) // 32 * 32, dtype=torch.float64)
    v[:, :c] = x
    v = v.view(n, -1, 32)
    top = v.abs().amax(-1, keepdim=True)
    low, high = (-120, 121) if fmt == "int8" else (-110, 119)
    fits = (lambda s: torch.round(top / power(s)) <= 127) if fmt == "int8" else (lambda s: top / power(s) <= 448)
    s = torch.full_like(top, low)
    for _ in range(high - low):
        s = torch.where(fits(s) | (s >= high), s, s + 1)
    w = v / power(s)
    if fmt == "int8":
        q = torch.round(w).clamp(-127, 127)
    else:
        _, e = torch.frexp(w.abs().clamp(min=2.0 ** -6))
        step = power(e.double() - 4)
        q = (torch.round(w / step) * step).clamp(-448, 448)
    out = q * power(s)
    out[~torch.isfinite(top).expand_as(out)] = float("nan")
    return out.view(n, -1)[:, :c]


def rows(n, c, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, c, generator=g) * torch.exp(2 * torch.randn(1, c, generator=g))
    x[torch.rand(n, c, generator=g) < 0.3] = 0
    return x.to(dtype).cuda()


DTYPES = [torch.float32, torch.bfloat16]
FMTS = ["int8", "e4m3"]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,c", [(1, 1), (1, 32), (7, 16), (33, 20), (5, 31), (64, 64), (129, 100), (3, 333), (2, 4096), (300, 8)])
def test_restored_values_are_the_definition(act8, n, c, dtype, fmt):
    x = rows(n, c, dtype, n * 1000 + c)
    held = act8.hold(x, fmt)
    assert held.codes.shape == (n, act8.pitch(c)) and held.scales.shape == (n, act8.pitch(c) // 32)
    assert held.nbytes() == held.codes.numel() + held.scales.numel()
    want = restored(x, fmt)
    for out_type in DTYPES:  # exact in either type
        got = held.restore(out_type)
        assert got.dtype == out_type and torch.equal(got.cpu().double(), want)
    assert held.restore().dtype == dtype
    assert not held.codes[:, c:].any()  # zero codes behind the last channel
    off = (want - x.cpu().double()).abs()
    pad = torch.zeros(n, act8.pitch(c), dtype=torch.float64)
    pad[:, :c] = x.cpu().double().abs()
    top = pad.view(n, -1, 32).amax(-1).repeat_interleave(32, 1)[:, :c]
    if fmt == "int8":
        assert (off <= top / 127.5).all()
    else:
        assert (off <= torch.maximum(x.cpu().double().abs() * 2.0 ** -4, top * 2.0 ** -17)).all()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_borders_of_the_codes(act8, dtype, fmt):
    """ties, the values where the exponent changes, the smallest and the largest numbers, zeros"""
    v = [0.0, 1.0, 127.0, 127.5, 127.25, 126.5, 128.0, 255.0, 254.0, 448.0, 449.0, 464.0, 480.0, 2.0 ** -9, 2.0 ** -10, 3 * 2.0 ** -11,
         1e-30, 1e-38, 1e-44, 3.3e38, 3.0e38, 2.0 ** 127, 0.875, 0.4375, 1.75, 1.7578125]
    x = torch.zeros(len(v) * 2, 40)
    for i, a in enumerate(v):
        x[2 * i, i % 32] = a
        x[2 * i + 1, :32] = torch.linspace(-1, 1, 32) * a
        x[2 * i + 1, 39] = -a
    x = x.to(dtype).cuda()
    assert torch.equal(act8.hold(x, fmt).restore(torch.float32).cpu().double(), restored(x, fmt))
    assert torch.isfinite(act8.hold(x, fmt).restore(torch.float32)).all()


@pytest.mark.parametrize("fmt", FMTS)
def test_non_finite_values_make_their_group_nan(act8, fmt):
    x = rows(6, 96, torch.float32)
    x[1, 40], x[2, 0], x[4, 95] = float("inf"), float("nan"), float("-inf")
    got = act8.hold(x, fmt).restore().cpu()
    bad = torch.zeros(6, 3, dtype=torch.bool)
    bad[1, 1] = bad[2, 0] = bad[4, 2] = True
    assert torch.equal(torch.isnan(got), bad.repeat_interleave(32, 1))
    assert torch.equal(got.double()[~torch.isnan(got)], restored(x, fmt)[~torch.isnan(got)])


@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts(act8, dtype):
    """rows at a distance, a start in the middle of a vector, transposed and expanded rows, an output inside a larger matrix"""
    big = rows(50, 130, dtype)
    for x in (big[:, :64], big[3:40, 1:65], big[::3, 2:100], big.t(), big[:1, :32].expand(9, 32), big[5:6, 7:20]):
        held = act8.hold(x, "int8")
        want = restored(x, "int8")
        assert torch.equal(held.restore().cpu().double(), want)
        n, c = x.shape
        room = torch.full((n + 2, c + 9), 7.0, dtype=dtype, device="cuda")
        out = room[1:n + 1, 3:c + 3]
        assert held.restore(out=out) is out
        assert torch.equal(out.cpu().double(), want)
        out.fill_(7.0)
        assert (room == 7.0).all()  # nothing around it was touched
    assert act8.hold(big[:0], "e4m3").restore().shape == (0, 130)


def test_offsets_beyond_32_bits(act8):
    n, c = (1 << 22) + 5, 520  # 2.2e9 values
    x = torch.zeros((n, c), dtype=torch.bfloat16, device="cuda")
    x[-3:] = rows(3, c, torch.bfloat16)
    held = act8.hold(x, "int8")
    out = held.restore()
    assert torch.equal(out[-3:].cpu().double(), restored(x[-3:], "int8")) and not out[:4].any()
    dy = torch.zeros((n, 8), dtype=torch.bfloat16, device="cuda")
    dy[-3:] = 1
    want = restored(x[-3:], "int8").sum(0)
    assert torch.allclose(act8.weight_grad(held, dy)[:, 0].cpu().double(), want, rtol=4 * EPS32, atol=4 * EPS32 * float(want.abs().max()))


def table(n_in, n_out, kvol, density, seed):
    g = torch.Generator().manual_seed(seed)
    nbr = torch.randint(0, max(n_in, 1), (kvol, n_out), generator=g)
    nbr[torch.rand(kvol, n_out, generator=g) >= density] = -1
    return nbr.to(torch.int32)


def reference_dw(x64, dy, nbr):
    """(dw, the sums of the absolute products) in 64 bits on the CPU"""
    dy = dy.cpu().double()
    if nbr is None:
        return x64.t() @ dy, x64.abs().t() @ dy.abs()
    dw, mag = [], []
    for k in range(nbr.shape[0]):
        i = nbr[k, :dy.shape[0]].cpu().long()
        o = torch.nonzero((i >= 0) & (i < x64.shape[0]))[:, 0]
        dw.append(x64[i[o]].t() @ dy[o])
        mag.append(x64[i[o]].abs().t() @ dy[o].abs())
    return torch.stack(dw), torch.stack(mag)


def check_dw(got, x64, dy, nbr):
    want, mag = reference_dw(x64, dy, nbr)
    # every product is rounded at most once (float32 dy in three bf16 terms: 2^-25), then at most n additions
    tol = (dy.shape[0] + 4) * EPS32 * mag
    assert got.dtype == torch.float32 and got.shape == want.shape
    off = (got.cpu().double() - want).abs()
    assert (off <= tol).all(), float((off - tol).max())


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,cin,cout", [(1, 1, 1), (1, 64, 64), (5, 3, 7), (63, 16, 16), (64, 32, 64), (65, 100, 36), (129, 33, 130),
                                        (200, 256, 40), (70, 40, 300), (300, 128, 128), (31, 520, 8)])
def test_weight_gradient_of_a_linear_layer(act8, n, cin, cout, dtype, fmt):
    x, dy = rows(n, cin, dtype, 1), rows(n, cout, dtype, 2)
    got = act8.weight_grad(act8.hold(x, fmt), dy)
    check_dw(got, restored(x, fmt), dy, None)
    assert torch.equal(got, act8.weight_grad(act8.hold(x, fmt), dy))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n_in,n_out,kvol,cin,cout,density", [
    (300, 300, 27, 16, 16, 0.5), (100, 260, 27, 32, 64, 0.3), (257, 190, 3, 64, 64, 0.7), (64, 64, 27, 128, 128, 0.5),
    (50, 50, 5, 24, 20, 0.5), (40, 700, 8, 7, 9, 1.0), (90, 90, 27, 64, 64, 0.0), (1, 1, 27, 64, 32, 1.0), (33, 129, 1, 16, 48, 0.6)])
def test_weight_gradient_through_a_table(act8, n_in, n_out, kvol, cin, cout, density, dtype):
    x, dy = rows(n_in, cin, dtype, 3), rows(n_out, cout, dtype, 4)
    nbr = table(n_in, n_out, kvol, density, n_in + n_out)
    got = act8.weight_grad(act8.hold(x, "int8"), dy, nbr.cuda())
    check_dw(got, restored(x, "int8"), dy, nbr)


def test_table_rows_behind_the_last_and_entries_out_of_range(act8):
    """a table longer than dy, entries below zero and behind the last held row: all absent; the same row many times"""
    x, dy = rows(40, 64, torch.float32, 5), rows(100, 64, torch.float32, 6)
    nbr = table(40, 170, 9, 0.6, 7)
    nbr[0, :50] = 40
    nbr[1, :50] = 2 ** 31 - 1
    nbr[2, :50] = -(2 ** 31)
    nbr[3, :] = 11
    nbr[:, 100:] = 3
    got = act8.weight_grad(act8.hold(x, "e4m3"), dy, nbr.cuda())
    check_dw(got, restored(x, "e4m3"), dy, nbr)
    assert not act8.weight_grad(act8.hold(x[:0], "int8"), dy, nbr.cuda()).any()
    assert not act8.weight_grad(act8.hold(x, "int8"), dy[:0], nbr.cuda()).any()


def test_the_rulebook_of_a_layer(act8):
    """against the framework's own weight gradient of a submanifold layer on the restored rows"""
    from det3d_amd import _lib, spconv

    g = torch.Generator().manual_seed(1)
    cells = torch.randperm(12 * 20 * 20, generator=g)[:1500].sort().values
    idx = torch.stack([torch.zeros_like(cells), cells // 400, cells // 20 % 20, cells % 20], 1).int().cuda()
    conv = spconv.SubMConv3d(64, 64, 3, bias=False, indice_key="k").cuda()
    x, dy = rows(1500, 64, torch.bfloat16, 8), rows(1500, 64, torch.bfloat16, 9)
    held = act8.hold(x, "int8")
    feats = held.restore().requires_grad_()
    y = conv(spconv.SparseConvTensor(feats, idx, [12, 20, 20], 1))
    (want,) = torch.autograd.grad(y.features, conv.weight, dy)
    rb = y.indice_dict["k"]
    got = act8.weight_grad(held, dy, rb.nbr_out.view(rb.kvol, rb.cap_out))
    _, mag = reference_dw(restored(x, "int8"), dy, rb.nbr_out.view(rb.kvol, rb.cap_out))
    assert ((got.cpu() - want.view_as(got).cpu()).abs().double() <= 2 * 1504 * EPS32 * mag).all()
    assert _lib.lib().d3d_act8_pitch(64) == 64


@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts_of_dy(act8, dtype):
    x = rows(90, 48, dtype, 1)
    held = act8.hold(x, "int8")
    big = rows(200, 131, dtype, 2)
    for dy in (big[:90, :64], big[5:95, 3:67], big[::2, 1:100][:90], big.t()[:90], big[:90, 130:]):
        check_dw(act8.weight_grad(held, dy), restored(x, "int8"), dy, None)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cout", [2, 6, 9, 12, 15, 31, 33, 63, 65, 100, 127, 129, 257, 263])
def test_widths_of_dy(act8, cout, dtype):
    """widths that end inside a vector, with other values in front of the first row and behind the last, and between the rows"""
    x = rows(150, 40, dtype, 1)
    held = act8.hold(x, "int8")
    big = torch.full((152, cout + 3), float("nan"), dtype=dtype, device="cuda")
    big[1:151, 1:cout + 1] = rows(150, cout, dtype, 2)
    check_dw(act8.weight_grad(held, big[1:151, 1:cout + 1]), restored(x, "int8"), big[1:151, 1:cout + 1], None)
    nbr = table(150, 150, 5, 0.6, cout)
    check_dw(act8.weight_grad(held, big[1:151, 1:cout + 1], nbr.cuda()), restored(x, "int8"), big[1:151, 1:cout + 1], nbr)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_non_finite_groups_reach_the_gradient(act8, dtype, fmt):
    """a group that is restored as NaN makes NaN of its 32 channels, and of the offsets that meet its row only"""
    x, dy = rows(70, 96, dtype, 1), rows(70, 33, dtype, 2)
    dy[9].fill_(1.0)
    x[9, 40], x[9, 95] = float("inf"), float("nan")
    bad = torch.zeros(96, dtype=torch.bool)
    bad[32:] = True
    dw = act8.weight_grad(act8.hold(x, fmt), dy).cpu()
    assert torch.isnan(dw[bad]).all() and torch.isfinite(dw[~bad]).all()
    nbr = torch.arange(70).repeat(3, 1).int()
    nbr[1][nbr[1] == 9] = -1  # (an absent neighbour)
    dw = act8.weight_grad(act8.hold(x, fmt), dy, nbr.cuda()).cpu()
    assert torch.isnan(dw[0][bad]).all() and torch.isnan(dw[2][bad]).all() and torch.isfinite(dw[1]).all()
    assert torch.isfinite(dw[:, ~bad]).all()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_largest_and_smallest_rows_through_the_gradient(act8, dtype, fmt):
    """groups at both ends of the scales' range: a restored value is finite and meets dy as it is"""
    x, dy = rows(130, 64, dtype, 1), rows(130, 16, dtype, 2)
    x = x / x.abs().amax()
    x[:65, :32] *= 3.3e38
    x[65:, 32:] *= 1e-28
    dy[:65] *= 1e-25
    held = act8.hold(x, fmt)
    assert torch.isfinite(held.restore()).all()
    check_dw(act8.weight_grad(held, dy), restored(x, fmt), dy, None)


def test_non_finite_gradients_are_seen(act8):
    x, dy = rows(70, 64, torch.float32, 1), rows(70, 64, torch.float32, 2)
    dy[3, 5] = float("nan")
    dw = act8.weight_grad(act8.hold(x, "int8"), dy)
    assert torch.isnan(dw[:, 5]).all() and torch.isfinite(dw[:, :5]).all() and torch.isfinite(dw[:, 6:]).all()
    dy[3, 5] = 0
    x[7, 40] = float("inf")
    dw = act8.weight_grad(act8.hold(x, "int8"), dy)
    assert torch.isnan(dw[32:]).all() and torch.isfinite(dw[:32]).all()


def test_on_another_stream_and_in_a_graph(act8):
    x, dy = rows(500, 64, torch.float32, 1), rows(500, 64, torch.float32, 2)
    nbr = table(500, 500, 27, 0.5, 1).cuda()
    step = lambda: act8.weight_grad(act8.hold(x, "int8"), dy, nbr)  # noqa: E731
    want = step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = step()
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        a = step()
    with torch.cuda.graph(g2):  # two graphs do not share a workspace
        b = step()
    for k in range(4):
        x.copy_(rows(500, 64, torch.float32, 10 + k))
        want = step()
        g1.replay()
        g2.replay()
        g1.replay()
        torch.cuda.synchronize()
        assert torch.equal(a, want) and torch.equal(b, want)


def test_two_at_once(act8):
    """the same held rows read on two streams at the same time, each call with a workspace of its own"""
    x, dy = rows(3000, 64, torch.float32, 1), [rows(3000, 64, torch.float32, 2 + k) for k in range(2)]
    held, nbr = act8.hold(x), table(3000, 3000, 27, 0.5, 1).cuda()
    want = [act8.weight_grad(held, d, nbr) for d in dy]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(act8.weight_grad(held, dy[k], nbr))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[k]) for k in range(2) for g in got[k])


def test_refusals(act8):
    from det3d_amd._lib import D3dError

    x, dy = rows(10, 32, torch.float32), rows(10, 8, torch.float32)
    held = act8.hold(x)
    with pytest.raises(ValueError, match="format"):
        act8.hold(x, "int4")
    with pytest.raises(D3dError, match="float32 / bfloat16"):
        act8.hold(x.half())
    with pytest.raises(D3dError, match="rows"):
        act8.hold(x[0])
    with pytest.raises(D3dError, match="GPU only"):
        act8.hold(x.cpu())
    with pytest.raises(D3dError, match="no channels"):
        act8.hold(x[:, :0])
    with pytest.raises(D3dError, match="float32 / bfloat16"):
        held.restore(torch.float16)
    with pytest.raises(D3dError, match="out must be"):
        held.restore(out=torch.empty(10, 33, device="cuda"))
    with pytest.raises(D3dError, match="out must be"):
        held.restore(out=torch.empty(1, 32, device="cuda").expand(10, 32))
    with pytest.raises(D3dError, match="no table"):
        act8.weight_grad(held, dy[:9])
    with pytest.raises(D3dError, match="int32"):
        act8.weight_grad(held, dy, torch.zeros(3, 10, dtype=torch.int64, device="cuda"))
    with pytest.raises(D3dError, match="int32"):
        act8.weight_grad(held, dy, torch.zeros(10, 3, dtype=torch.int32, device="cuda").t())
    with pytest.raises(D3dError, match="table of"):
        act8.weight_grad(held, dy, torch.zeros(3, 9, dtype=torch.int32, device="cuda"))


def test_a_rewound_arena_is_noticed(act8):
    from det3d_amd import arena

    a = arena.BumpArena("cuda", "t", 1 << 20).begin()
    with arena.bound(a):
        held = act8.hold(rows(4, 32, torch.float32))
    held.restore()
    a.begin()
    with pytest.raises(arena.ArenaError):
        held.restore()
    with pytest.raises(arena.ArenaError):
        act8.weight_grad(held, rows(4, 8, torch.float32))


@pytest.mark.parametrize("n,kvol,cin", [(1, 1, 16), (64, 1, 64), (63, 3, 16), (128, 27, 16), (640, 5, 64), (4096, 27, 32), (8129, 3, 48)])
def test_tables_that_end_with_their_buffer(act8, n, kvol, cin):
    """the entries requested ahead of the rows end with the table: the last offset's rows are all there, and nothing behind them counts"""
    x, dy = rows(n, cin, torch.bfloat16, 1), rows(n, 16, torch.bfloat16, 2)
    nbr = table(n, n, kvol, 0.5, n)
    nbr[-1] = torch.arange(n, dtype=torch.int32).flip(0)
    check_dw(act8.weight_grad(act8.hold(x, "int8"), dy, nbr.cuda()), restored(x, "int8"), dy, nbr)


def test_small_gradients(act8):
    """dy down to the smallest numbers: the three bfloat16 terms leave at most 2^-134 of a value (half of bfloat16's smallest step),
    and a sum below the normal numbers is rounded to 2^-149 at every addition"""
    x = rows(64, 40, torch.float32, 1)
    g = torch.Generator().manual_seed(5)
    dy = (1 + torch.rand(64, 24, generator=g)) * torch.exp2(-100 - torch.randint(0, 45, (64, 24), generator=g).float())
    x64 = restored(x, "int8")
    got = act8.weight_grad(act8.hold(x), dy.cuda())
    want, mag = reference_dw(x64, dy, None)
    tol = 68 * EPS32 * mag + 2.0 ** -134 * x64.abs().sum(0)[:, None] + 3 * 64 * 2.0 ** -149
    assert ((got.cpu().double() - want).abs() <= tol).all()
    exact = dy.abs() >= 2.0 ** -110
    one = torch.zeros(64, 40)
    one[:, 0] = 1
    dy1 = torch.where(exact, dy, torch.zeros(()))
    for r in range(0, 64, 16):  # one row alone: the value itself
        single = torch.zeros_like(dy1)
        single[r] = dy1[r]
        assert torch.equal(act8.weight_grad(act8.hold(one.cuda()), single.cuda())[0].cpu(), single[r])
