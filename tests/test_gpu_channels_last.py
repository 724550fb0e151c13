"""group_norm_act and linear_act on the GPU against plain 64-bit forms (tests/channels_last.py
has the formulas and says how the bounds are derived)."""
from __future__ import annotations

import pytest

import s2b200

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

import channels_last as cl  # noqa: E402

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
NORM_TYPES = [(F16, F16), (BF16, BF16), (F32, F32), (F32, F16), (F32, BF16)]


@pytest.fixture(scope="module", autouse=True)
def device():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    assert s2b200.device_check(0) == 0, s2b200.last_error()


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(shape, gen, dtype=F32):
    return torch.randn(shape, generator=gen, device="cuda").to(dtype)


def _features(shape, gen, dtype, pad=0):
    C = shape[-1]
    x = _normal(shape[:-1] + (C + pad,), gen)[..., :C]
    return (x * torch.exp(0.5 * _normal((C,), gen)) + 2 * _normal((C,), gen)).to(dtype)


def _padded(x, pad):
    """x in rows of `pad` values more, NaN in them."""
    big = torch.full(x.shape[:-1] + (x.shape[-1] + pad,), float("nan"), dtype=x.dtype, device=x.device)
    big[..., :x.shape[-1]] = x
    return big, big[..., :x.shape[-1]]


# ---- group norm ------------------------------------------------------------------

# (samples, positions, channels, groups): single values, one channel a group, groups that no vector
# fits, blocks of columns (more channels than a block's threads hold), few and many rows
NORM_SHAPES = [(1, 1, 1, 1), (1, 1, 32, 32), (2, 1, 64, 8), (1, 2, 8, 1), (2, 7, 96, 32), (3, 1000, 130, 10),
               (2, 257, 512, 32), (5, 64, 40, 8), (1, 5003, 24, 8), (1, 17, 4104, 3), (2, 33, 8192, 2),
               (1, 9, 2056, 257), (1, 40, 1024, 1024), (1, 3001, 128, 1), (17, 130, 48, 16), (1, 70001, 16, 2),
               (2, 14400, 64, 32)]


@pytest.mark.parametrize("types", NORM_TYPES, ids=lambda t: f"{t[0]}-{t[1]}".replace("torch.", ""))
@pytest.mark.parametrize("shape", NORM_SHAPES, ids=str)
def test_norm_shapes(shape, types):
    S, P, C, G = shape
    gen = _gen(P + C)
    x = _features((S, P, C), gen, types[0])
    w, b = 1 + 0.1 * _normal((C,), gen), 0.1 * _normal((C,), gen)
    act = cl.ACTS[(P + C + G) % 5]
    y = s2b200.group_norm_act(x, G, w, b, eps=1e-6, activation=act, out_dtype=types[1])
    assert y.dtype == types[1] and y.shape == x.shape
    cl.check(y, *cl.norm_exact(x, G, w, b, 1e-6, act), f"{shape} {act}")


@pytest.mark.parametrize("act", cl.ACTS)
@pytest.mark.parametrize("affine", [(False, False), (True, False), (False, True)])
def test_norm_activations_and_affine(act, affine):
    gen = _gen(3)
    x = _features((2, 300, 64), gen, F16)
    w = _normal((64,), gen) if affine[0] else None
    b = _normal((64,), gen) if affine[1] else None
    y = s2b200.group_norm_act(x, 16, w, b, eps=1e-5, activation=act)
    cl.check(y, *cl.norm_exact(x, 16, w, b, 1e-5, act))


@pytest.mark.parametrize("types", NORM_TYPES, ids=lambda t: f"{t[0]}-{t[1]}".replace("torch.", ""))
@pytest.mark.parametrize("pads", [(8, 8), (0, 8), (8, 0), (1, 0), (0, 3), (2, 2), (4, 4), (5, 16)])
def test_norm_pitches(types, pads):
    """Rows of other pitches in and out; what lies between the rows is neither read nor written."""
    gen = _gen(4)
    x = _features((3, 211, 96), gen, types[0])
    _, xp = _padded(x, pads[0])
    buf, out = _padded(torch.zeros(3, 211, 96, dtype=types[1], device="cuda"), pads[1])
    w = 1 + 0.1 * _normal((96,), gen)
    r = s2b200.group_norm_act(xp, 32, w, None, activation="silu", out=out)
    assert r is out
    cl.check(out, *cl.norm_exact(x, 32, w, None, 1e-6, "silu"))
    assert torch.isnan(buf[..., 96:]).all()


def test_norm_frames_of_a_video():
    """[T, H, W, C] with the frames cut out of a longer clip: the sample stride is its own."""
    gen = _gen(5)
    clip = _features((6, 9, 11, 64), gen, BF16)
    x = clip[::2]
    y = s2b200.group_norm_act(x, 32, activation="silu")
    assert y.shape == x.shape and y.is_contiguous()
    cl.check(y, *cl.norm_exact(x, 32, None, None, 1e-6, "silu"))


@pytest.mark.parametrize("offset", [0, 1, 2, 4])
def test_norm_base_alignment(offset):
    gen = _gen(6)
    flat = _features((1, 1, 2 * 150 * 64 + 8), gen, F16).flatten()
    x = flat[offset:offset + 2 * 150 * 64].view(2, 150, 64)
    y = s2b200.group_norm_act(x, 32, activation="gelu_tanh")
    cl.check(y, *cl.norm_exact(x, 32, None, None, 1e-6, "gelu_tanh"))


@pytest.mark.parametrize("shape", [(2, 301, 64, 32), (1, 9000, 512, 32), (3, 50, 33, 11)])
@pytest.mark.parametrize("dtype", [F16, F32])
def test_norm_in_place(shape, dtype):
    S, P, C, G = shape
    x = _features((S, P, C), _gen(7), dtype)
    want = s2b200.group_norm_act(x, G, activation="silu")
    got = x.clone()
    s2b200.group_norm_act(got, G, activation="silu", out=got)
    assert torch.equal(got, want)


def test_norm_into_the_other_half_of_its_rows():
    """x and out are column ranges of one buffer."""
    gen = _gen(8)
    buf = _features((2, 77, 128), gen, F16)
    x = buf[..., :64].clone()
    s2b200.group_norm_act(buf[..., :64], 8, out=buf[..., 64:])
    assert torch.equal(buf[..., :64], x)
    cl.check(buf[..., 64:], *cl.norm_exact(x, 8, None, None, 1e-6, "none"))


@pytest.mark.parametrize("P", [40, 1000, 30000])
def test_norm_keeps_a_small_spread_about_a_large_mean(P):
    gen = _gen(9)
    x = 1000 + 0.5 * _normal((2, P, 64), gen)
    y = s2b200.group_norm_act(x, 8)
    cl.check(y, *cl.norm_exact(x, 8, None, None, 1e-6, "none"))


@pytest.mark.parametrize("at", [0, 1, 37, 4999])
def test_norm_with_an_outlier(at):
    """One value 10^4 spreads away, at the start of a run too: the other values keep their digits."""
    gen = _gen(10)
    x = _normal((1, 5000, 32), gen)
    x[0, at, 5] = 1e4
    y = s2b200.group_norm_act(x, 4)
    cl.check(y, *cl.norm_exact(x, 4, None, None, 1e-6, "none"))


def test_norm_of_equal_values():
    x = torch.full((2, 100, 32), 3.25, device="cuda", dtype=F16)
    b = torch.linspace(-1, 1, 32, device="cuda")
    y = s2b200.group_norm_act(x, 4, None, b)
    assert torch.equal(y, b.half().expand_as(y))


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("at", [0, 500])
def test_norm_bad_values_stay_in_their_group(bad, at):
    gen = _gen(11)
    x = _features((2, 1001, 32), gen, F16)
    y0 = s2b200.group_norm_act(x, 8, activation="relu")
    x[1, at, 9] = bad
    y = s2b200.group_norm_act(x, 8, activation="relu")
    assert torch.isnan(y[1, :, 8:12]).all()
    y[1, :, 8:12] = y0[1, :, 8:12]
    assert torch.equal(y, y0)


def test_norm_of_nothing():
    for shape in ((0, 5, 32), (3, 0, 32)):
        y = s2b200.group_norm_act(torch.empty(shape, device="cuda", dtype=F16), 8)
        assert y.shape == shape


@pytest.mark.parametrize("dtype", [F16, F32], ids=str)
@pytest.mark.parametrize("shape", [(3, 20000, 96), (2, 40000, 512), (4, 60000, 128), (2, 1500, 512), (1, 60000, 130),
                                   (40, 500, 640), (300, 64, 512), (1, 300000, 64), (2, 140000, 512)], ids=str)
def test_norm_gives_the_same_bits(shape, dtype):
    """Whatever the blocks' order: the joins' and the ring's hand-overs, many times over."""
    x = _features(shape, _gen(12), dtype)
    G = 10 if shape[2] == 130 else 32
    first = s2b200.group_norm_act(x, G, activation="silu")
    cl.check(first[:1], *cl.norm_exact(x[:1], G, None, None, 1e-6, "silu"))
    off = torch.zeros((), dtype=torch.int64, device="cuda")
    for _ in range(100):
        off += (s2b200.group_norm_act(x, G, activation="silu") != first).sum()
    assert off.item() == 0


@pytest.mark.parametrize("shape", [(1, 600000, 64, 32), (2, 300000, 128, 32), (1, 120000, 512, 32), (1, 2000000, 16, 4)])
def test_norm_of_large_samples(shape):
    """Samples beyond a block's, a cluster's and the chip's memory."""
    S, P, C, G = shape
    x = _features((S, P, C), _gen(13), BF16)
    y = s2b200.group_norm_act(x, G, activation="silu")
    for s in range(S):
        cl.check(y[s:s + 1], *cl.norm_exact(x[s:s + 1], G, None, None, 1e-6, "silu"))


# channels a group that make 1, 2, 4 and 8 moments of a vector, few and many groups, units that a ring of
# one pass, of several and of none to spare holds
@pytest.mark.parametrize("types", NORM_TYPES, ids=lambda t: f"{t[0]}-{t[1]}".replace("torch.", ""))
@pytest.mark.parametrize("shape", [(2, 40001, 256, 32), (3, 50000, 128, 32), (1, 300017, 64, 32), (9, 30011, 96, 32),
                                   (2, 60000, 192, 64), (1, 33000, 2048, 1), (1, 260001, 80, 16), (2, 150001, 512, 32)],
                         ids=str)
def test_norm_of_large_packed_units(shape, types):
    S, P, C, G = shape
    x = _features((S, P, C), _gen(P), types[0])
    w, b = 1 + 0.1 * _normal((C,), _gen(1)), 0.1 * _normal((C,), _gen(2))
    act = cl.ACTS[(P + C) % 5]
    y = s2b200.group_norm_act(x, G, w, b, activation=act, out_dtype=types[1])
    for s in range(S):
        cl.check(y[s:s + 1], *cl.norm_exact(x[s:s + 1], G, w, b, 1e-6, act), f"{shape} {act}")


@pytest.mark.parametrize("types", NORM_TYPES, ids=lambda t: f"{t[0]}-{t[1]}".replace("torch.", ""))
@pytest.mark.parametrize("shape,pad", [((2, 40001, 256, 32), 3), ((1, 50000, 130, 10), 0), ((2, 30000, 640, 32), 8),
                                       ((3, 60000, 64, 16), 8), ((1, 9000, 5120, 2), 0), ((10, 20000, 128, 32), 1)], ids=str)
def test_norm_of_large_units_in_pitched_rows(shape, pad, types):
    S, P, C, G = shape
    x = _features((S, P, C), _gen(P), types[0], pad)
    y = s2b200.group_norm_act(_padded(x, pad)[1], G, activation="gelu", out_dtype=types[1])
    for s in range(S):
        cl.check(y[s:s + 1], *cl.norm_exact(x[s:s + 1], G, None, None, 1e-6, "gelu"), f"{shape}")


@pytest.mark.parametrize("shape", [(2, 40000, 512, 32), (1, 400000, 64, 32), (2, 60001, 130, 10)], ids=str)
@pytest.mark.parametrize("dtype", [F16, F32], ids=str)
def test_norm_of_large_units_in_place(shape, dtype):
    S, P, C, G = shape
    x = _features((S, P, C), _gen(15), dtype)
    want = s2b200.group_norm_act(x, G, activation="silu")
    for _ in range(3):
        got = x.clone()
        s2b200.group_norm_act(got, G, activation="silu", out=got)
        assert torch.equal(got, want)


@pytest.mark.parametrize("shape", [(2, 40000, 512, 32), (1, 60001, 130, 10)], ids=str)
def test_norm_of_large_units_about_a_large_mean(shape):
    S, P, C, G = shape
    x = 300 + 0.5 * _normal((S, P, C), _gen(16))
    x[0, P // 3, 5] = 1e4
    y = s2b200.group_norm_act(x, G)
    for s in range(S):
        cl.check(y[s:s + 1], *cl.norm_exact(x[s:s + 1], G, None, None, 1e-6, "none"))


# Slices of the channels that the whole grid, or some of its blocks, hold at once: one block a slice and all of
# them, moments joined by each block for itself and by one for all, rows in one box and in two, 1 to 8 moments
# a vector, columns that do not fill the threads, last blocks with fewer rows.
SLICES = [(2, 1920, 512, 32), (40, 200, 1280, 32), (3, 57601, 512, 32), (1, 100003, 128, 32), (12, 9001, 320, 32),
          (20, 5003, 120, 24), (300, 64, 512, 32), (2000, 16, 512, 32), (7, 12007, 256, 1), (5, 6001, 640, 32),
          (9, 30011, 96, 24), (30, 1999, 208, 16)]


@pytest.mark.parametrize("types", NORM_TYPES, ids=lambda t: f"{t[0]}-{t[1]}".replace("torch.", ""))
@pytest.mark.parametrize("pads", [(0, 0), (8, 16)], ids=str)
@pytest.mark.parametrize("shape", SLICES, ids=str)
def test_norm_of_slices(shape, pads, types):
    S, P, C, G = shape
    gen = _gen(P + C)
    x = _padded(_features((S, P, C), gen, types[0]), pads[0])[1]
    buf, out = _padded(torch.zeros(S, P, C, dtype=types[1], device="cuda"), pads[1])
    w, b = 1 + 0.1 * _normal((C,), gen), 0.1 * _normal((C,), gen)
    act = cl.ACTS[(P + S + G) % 5]
    s2b200.group_norm_act(x, G, w, b, activation=act, out=out)
    for s in {0, S // 2, S - 1}:
        cl.check(out[s:s + 1], *cl.norm_exact(x[s:s + 1], G, w, b, 1e-6, act), f"{shape} {act}")
    assert torch.isnan(buf[..., C:]).all() and not torch.isnan(out).any()


@pytest.mark.parametrize("shape", SLICES, ids=str)
@pytest.mark.parametrize("dtype", [BF16, F32], ids=str)
def test_norm_of_slices_in_place(shape, dtype):
    S, P, C, G = shape
    x = _features((S, P, C), _gen(31), dtype)
    want = s2b200.group_norm_act(x, G, activation="silu")
    s2b200.group_norm_act(x, G, activation="silu", out=x)
    assert torch.equal(x, want)


@pytest.mark.parametrize("shape", [(2, 1920, 512, 32), (40, 200, 1280, 32), (3, 20001, 512, 32)], ids=str)
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_norm_of_slices_bad_values_and_equal_ones(shape, bad):
    S, P, C, G = shape
    x = _features(shape[:3], _gen(32), F16)
    y0 = s2b200.group_norm_act(x, G, activation="relu")
    k = C // G
    for at, g in ((0, 3), (P // 2, G - 1), (P - 1, 0)):
        z = x.clone()
        z[S - 1, at, g * k + 1] = bad
        y = s2b200.group_norm_act(z, G, activation="relu")
        assert torch.isnan(y[S - 1, :, g * k:(g + 1) * k]).all()
        y[S - 1, :, g * k:(g + 1) * k] = y0[S - 1, :, g * k:(g + 1) * k]
        assert torch.equal(y, y0)
    b = torch.linspace(-1, 1, C, device="cuda")
    y = s2b200.group_norm_act(torch.full(shape[:3], 3.25, device="cuda", dtype=F16), G, None, b)
    assert torch.equal(y, b.half().expand_as(y))


def test_norm_of_slices_about_a_large_mean():
    x = 1000 + 0.5 * _normal((2, 20000, 256), _gen(33))
    x[0, 777, 3] = 3e5
    y = s2b200.group_norm_act(x, 32)
    cl.check(y, *cl.norm_exact(x, 32, None, None, 1e-6, "none"))


def test_norm_of_slices_on_two_streams_and_replayed():
    """Two calls that need the whole grid each at the same time, eager and in graphs, on new inputs."""
    gen = _gen(34)
    xs = [_features((3, 20001, 512), gen, F16), _features((60, 300, 640), gen, F16)]
    want = [s2b200.group_norm_act(x, 32, activation="silu") for x in xs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    off = torch.zeros((), dtype=torch.int64, device="cuda")
    torch.cuda.synchronize()
    for _ in range(20):
        got = []
        for x, st in zip(xs, streams):
            with torch.cuda.stream(st):
                got.append(s2b200.group_norm_act(x, 32, activation="silu"))
        torch.cuda.synchronize()
        off += sum((g != w).sum() for g, w in zip(got, want))
    graphs = []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = s2b200.group_norm_act(x, 32, activation="silu")
        graphs.append((g, y))
    for x in xs:
        x.copy_(x.flip(0))
    want = [s2b200.group_norm_act(x, 32, activation="silu") for x in xs]
    torch.cuda.synchronize()
    for _ in range(5):
        for (g, _), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        off += sum((y != w).sum() for (_, y), w in zip(graphs, want))
    assert off.item() == 0


def test_norm_of_many_samples():
    x = _features((3000, 33, 48), _gen(17), F16)
    y = s2b200.group_norm_act(x, 16, activation="silu")
    cl.check(y, *cl.norm_exact(x, 16, None, None, 1e-6, "silu"))


def test_norm_past_2_31_values():
    S, P, C, G = 3, 5700000, 128, 32
    x = torch.empty((S, P, C), dtype=F16, device="cuda")
    gen = _gen(14)
    for s in range(S):
        x[s] = torch.randn((P, C), generator=gen, device="cuda", dtype=F16)
        x[s] += s
    y = s2b200.group_norm_act(x, G, activation="none")
    for s in range(S):
        var, mean = torch.zeros(G, dtype=torch.float64, device="cuda"), torch.zeros(G, dtype=torch.float64, device="cuda")
        for part in x[s].split(600000):
            mean += part.double().view(-1, G, C // G).sum(dim=(0, 2))
        mean /= P * (C // G)
        for part in x[s].split(600000):
            var += ((part.double().view(-1, G, C // G) - mean[:, None]) ** 2).sum(dim=(0, 2))
        sigma = (var / (P * (C // G)) + 1e-6).sqrt()
        for r0 in (0, P // 2, P - 1000):
            d = x[s, r0:r0 + 1000].double().view(-1, G, C // G) - mean[:, None]
            want = (d / sigma[:, None]).view(-1, C)
            room = ((d.abs() + mean.abs()[:, None]) / sigma[:, None]).view(-1, C) * 2.0 ** -17
            cl.check(y[s, r0:r0 + 1000], want, room)


# ---- matrix product ----------------------------------------------------------------

LINEAR_SHAPES = [(1, 1, 1), (1, 2560, 2560), (1, 777, 1001), (2, 16, 8), (3, 64, 5120), (7, 130, 65), (16, 128, 64),
                 (17, 100, 128), (33, 2560, 256), (58, 2560, 5120), (64, 96, 1000), (65, 320, 200), (100, 1, 512),
                 (128, 256, 1024), (129, 257, 72), (200, 513, 640), (300, 5, 24), (1237, 777, 1001), (1000, 2560, 512),
                 (4096, 256, 64), (4500, 515, 1032), (8200, 512, 1536), (20000, 24, 48)]


def _operands(M, N, K, dtype, seed, res=True, out_dtype=None):
    gen = _gen(seed)
    x, w = _normal((M, K), gen, dtype), (0.05 * _normal((N, K), gen)).to(dtype)
    b = _normal((N,), gen)
    r = _normal((M, N), gen, out_dtype or dtype) if res else None
    return x, w, b, r


@pytest.mark.parametrize("dtype", [F16, BF16], ids=str)
@pytest.mark.parametrize("shape", LINEAR_SHAPES, ids=str)
def test_linear_shapes(shape, dtype):
    M, N, K = shape
    x, w, b, r = _operands(M, N, K, dtype, M + N + K)
    act = cl.ACTS[(M + N) % 5]
    y = s2b200.linear_act(x, w, b, act, r)
    assert y.dtype == dtype and y.shape == (M, N)
    cl.check(y, *cl.linear_exact(x, w, b, act, r), f"{shape} {act}")


@pytest.mark.parametrize("act", cl.ACTS)
@pytest.mark.parametrize("parts", [(False, False), (True, False), (False, True), (True, True)])
@pytest.mark.parametrize("shape", [(1, 200, 96), (40, 264, 192), (700, 264, 192), (4300, 256, 1024)], ids=str)
def test_linear_epilogues(shape, act, parts):
    x, w, b, r = _operands(*shape, F16, 21)
    b, r = b if parts[0] else None, r if parts[1] else None
    cl.check(s2b200.linear_act(x, w, b, act, r), *cl.linear_exact(x, w, b, act, r))


@pytest.mark.parametrize("dtype", [F16, BF16], ids=str)
@pytest.mark.parametrize("shape", [(1, 300, 640), (50, 333, 640), (333, 200, 2560), (5000, 512, 1024)], ids=str)
def test_linear_fp32_out(shape, dtype):
    x, w, b, r = _operands(*shape, dtype, 22, out_dtype=F32)
    y = s2b200.linear_act(x, w, b, "silu", r, out_dtype=F32)
    assert y.dtype == F32
    cl.check(y, *cl.linear_exact(x, w, b, "silu", r))


@pytest.mark.parametrize("shape", [(1, 60, 72), (30, 120, 72), (500, 250, 200), (4200, 260, 1030)], ids=str)
@pytest.mark.parametrize("pads", [(8, 8, 8, 8), (1, 0, 0, 0), (0, 1, 0, 0), (0, 0, 1, 0), (0, 0, 0, 1), (3, 8, 2, 5)])
def test_linear_pitches(shape, pads):
    """x, w, residual and out in rows of other pitches; nothing between the rows counts or changes."""
    x, w, b, r = _operands(*shape, BF16, 23)
    xp, wp, rp = _padded(x, pads[0])[1], _padded(w, pads[1])[1], _padded(r, pads[2])[1]
    buf, out = _padded(torch.zeros_like(r), pads[3])
    s2b200.linear_act(xp, wp, b, "gelu", rp, out=out)
    cl.check(out, *cl.linear_exact(x, w, b, "gelu", r))
    assert torch.isnan(buf[..., shape[1]:]).all()


@pytest.mark.parametrize("shape", [(1, 64, 64), (60, 160, 96), (900, 160, 96), (4200, 256, 1024)], ids=str)
def test_linear_onto_its_residual(shape):
    x, w, b, r = _operands(*shape, F16, 24)
    want = s2b200.linear_act(x, w, b, "none", r)
    got = r.clone()
    s2b200.linear_act(x, w, b, "none", got, out=got)
    assert torch.equal(got, want)


@pytest.mark.parametrize("shape", [(9000, 512, 512), (20000, 300, 192), (70000, 128, 64)], ids=str)
@pytest.mark.parametrize("dtype", [F16, BF16], ids=str)
@pytest.mark.parametrize("out_dtype", [None, F32], ids=str)
def test_linear_of_short_sums_and_many_rows(shape, dtype, out_dtype):
    """The VAE's 1 x 1 projections: few products a sum, many rows."""
    x, w, b, r = _operands(*shape, dtype, 29, out_dtype=out_dtype)
    y = s2b200.linear_act(x, w, b, "silu", r, out_dtype=out_dtype)
    cl.check(y, *cl.linear_exact(x, w, b, "silu", r))


def test_linear_of_leading_dimensions():
    x, w, b, _ = _operands(60, 48, 64, F16, 25, res=False)
    y = s2b200.linear_act(x.view(3, 4, 5, 64), w, b, "relu")
    assert y.shape == (3, 4, 5, 48) and torch.equal(y.view(60, 48), s2b200.linear_act(x, w, b, "relu"))
    assert s2b200.linear_act(x[0], w, b, "relu").shape == (48,)
    assert s2b200.linear_act(x[:0], w, b).shape == (0, 48)


@pytest.mark.parametrize("shape", [(20, 130, 200), (1000, 130, 200), (4300, 256, 1024)], ids=str)
def test_linear_bad_rows_stay_alone(shape):
    """Infinite and NaN inputs reach their own row (x) or column (w) only."""
    x, w, b, r = _operands(*shape, F16, 26)
    y0 = s2b200.linear_act(x, w, b, "relu", r)
    x, w = x.clone(), w.clone()
    x[3, 7] = float("inf")
    w[5, 9] = float("nan")
    y = s2b200.linear_act(x, w, b, "relu", r)
    keep = torch.ones_like(y, dtype=torch.bool)
    keep[3], keep[:, 5] = False, False
    assert torch.equal(y[keep], y0[keep])
    assert torch.isnan(y[:, 5]).all()
    want = cl.linear_exact(x[3:4].float(), w.float(), b, "relu", r[3:4])[0]
    assert torch.equal(torch.isnan(y[3:4]), torch.isnan(want)) and torch.equal(torch.isinf(y[3:4]), torch.isinf(want))


@pytest.mark.parametrize("shape", [(1, 2560, 2560), (4, 300, 520), (58, 2560, 5120), (128, 640, 2560), (700, 500, 1024),
                                   (1237, 777, 1001), (5000, 512, 512), (4300, 2560, 1024)], ids=str)
@pytest.mark.parametrize("out_dtype", [None, F32], ids=str)
def test_linear_gives_the_same_bits(shape, out_dtype):
    """Whatever the blocks' order: the hand-overs of operands, sums, residuals and results, many times over."""
    x, w, b, r = _operands(*shape, F16, 27, out_dtype=out_dtype)
    first = s2b200.linear_act(x, w, b, "silu", r, out_dtype=out_dtype)
    off = torch.zeros((), dtype=torch.int64, device="cuda")
    for _ in range(60):
        off += (s2b200.linear_act(x, w, b, "silu", r, out_dtype=out_dtype) != first).sum()
    assert off.item() == 0


def test_linear_past_2_31_values():
    """Offsets of x, residual and y pass 2^31 elements."""
    M, N, K = 4300000, 512, 520
    gen = _gen(28)
    x = torch.empty((M, K), dtype=F16, device="cuda").normal_(generator=gen)
    w = (0.05 * _normal((N, K), gen)).half()
    r = torch.empty((M, N), dtype=F16, device="cuda").normal_(generator=gen)
    y = s2b200.linear_act(x, w, None, "none", r)
    for at in (0, M // 2, M - 500):
        rows = slice(at, at + 500)
        cl.check(y[rows], *cl.linear_exact(x[rows], w, None, "none", r[rows]))


# ---- streams, graphs, threads --------------------------------------------------------

def _calls(seed):
    gen = _gen(seed)
    x = _features((2, 6000, 64), gen, F16)
    wide = _features((1, 40000, 512), gen, F16)
    a, w, b, r = _operands(300, 264, 1000, F16, seed)
    one = a[:1]
    odd = _padded(a, 3)[1]

    def run(**kw):
        return [s2b200.group_norm_act(x, 32, activation="silu", **kw), s2b200.group_norm_act(wide, 32, **kw),
                s2b200.linear_act(a, w, b, "gelu", r, **kw), s2b200.linear_act(one, w, b, **kw),
                s2b200.linear_act(odd, w, b, "silu", **kw)]

    return (x, wide, a, one, odd, w, b, r), run


def test_other_streams():
    _, run = _calls(31)
    want = run()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    got = run(stream=side)
    side.synchronize()
    assert all(torch.equal(g, w) for g, w in zip(got, want))
    with torch.cuda.stream(side):
        got = run()
    side.synchronize()
    assert all(torch.equal(g, w) for g, w in zip(got, want))


def test_two_streams_at_once():
    data = [_calls(32), _calls(33)]
    want = [run() for _, run in data]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in data]
    got = [[], []]
    for _ in range(20):
        for i, (_, run) in enumerate(data):
            got[i].append(run(stream=streams[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for outs in got[i]:
            assert all(torch.equal(g, w) for g, w in zip(outs, want[i]))


def test_captured_and_replayed_on_new_inputs():
    (x, wide, a, one, odd, w, b, r), run = _calls(34)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        run()
    side.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = run()
        graphs.append((g, outs))
    for seed in (35, 36):
        gen = _gen(seed)
        for t in (x, wide, a, odd, r):
            t.copy_(_normal(t.shape, gen))
        want = run()
        for g, outs in graphs:
            g.replay()
        for g, outs in graphs:
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(outs, want))


def test_threads():
    import threading
    data = [_calls(37 + i) for i in range(4)]
    want = [run() for _, run in data]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        try:
            s = torch.cuda.Stream()
            for _ in range(10):
                got = data[i][1](stream=s)
                s.synchronize()
                if not all(torch.equal(g, w) for g, w in zip(got, want[i])):
                    bad.append(i)
        except Exception as e:  # noqa: BLE001
            bad.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad, bad


# ---- together ------------------------------------------------------------------------

@pytest.mark.parametrize("C,frames,H,W", [(512, 2, 12, 20), (256, 1, 9, 13)])
def test_vae_mid_block_attention_channels_last(C, frames, H, W):
    """Norm -> q, k, v projections -> the spatial attention core -> output projection + residual:
    the VAE's mid-block attention on token-major fp16, against 64 bits. Roundings to fp16 on the
    way: the norm, q, k, v, the probabilities, the attention and the result (the last one is
    check()'s own), 2^-11 relative each; a softmax over scores of size s turns a relative error of
    q and k into s times as much, s = 4 at most here: the branch is off by 16 * 2^-11 of its size."""
    gen = _gen(41)
    tokens = H * W
    x = _features((frames, tokens, C), gen, F16)
    gw, gb = 1 + 0.1 * _normal((C,), gen), 0.1 * _normal((C,), gen)
    ws = [(_normal((C, C), gen) * C ** -0.5).half() for _ in range(4)]
    bs = [0.1 * _normal((C,), gen) for _ in range(4)]
    h = s2b200.group_norm_act(x, 32, gw, gb)
    q, k, v = (s2b200.linear_act(h, w, b).view(-1, C) for w, b in zip(ws[:3], bs))
    o = torch.empty_like(q)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    s2b200.spatial_attention(q, k, v, C, frames, tokens, o, err)
    y = s2b200.linear_act(o.view_as(x), ws[3], bs[3], residual=x, err=err)
    assert err.item() == 0
    h64 = cl.norm_exact(x, 32, gw, gb, 1e-6, "none")[0]
    q64, k64, v64 = (h64 @ w.double().t() + b.double() for w, b in zip(ws[:3], bs))
    scores = q64 @ k64.transpose(1, 2) * C ** -0.5
    branch = torch.softmax(scores, dim=-1) @ v64 @ ws[3].double().t() + bs[3].double()
    size = branch.abs().mean() + branch.abs()
    cl.check(y, x.double() + branch, 16 * 2.0 ** -11 * size)


def test_timestep_mlp():
    """One row through silu, silu and a wide projection (the timestep embedding's MLP): each layer
    against 64 bits of its own input."""
    gen = _gen(42)
    t = _normal((1, 256), gen, BF16)
    dims = (256, 2560, 2560, 15360)
    for i, act in enumerate(("silu", "silu", "none")):
        w = (_normal((dims[i + 1], dims[i]), gen) * dims[i] ** -0.5).to(BF16)
        b = 0.1 * _normal((dims[i + 1],), gen)
        out = s2b200.linear_act(t, w, b, act)
        cl.check(out, *cl.linear_exact(t, w, b, act, None))
        t = out


def test_wrappers_refuse_what_they_cannot_run():
    x = torch.zeros(4, 64, dtype=F16, device="cuda")
    w = torch.zeros(32, 64, dtype=F16, device="cuda")
    v = torch.zeros(64, device="cuda")
    grad = x.float().half().requires_grad_()
    calls = [
        lambda: s2b200.group_norm_act(x, 7), lambda: s2b200.group_norm_act(x[0], 8),
        lambda: s2b200.group_norm_act(x, 8, activation="swish"), lambda: s2b200.group_norm_act(x, 8, v.half()),
        lambda: s2b200.group_norm_act(x, 8, v[:32]), lambda: s2b200.group_norm_act(x, 8, v.cpu()),
        lambda: s2b200.group_norm_act(x, 8, torch.zeros(128, device="cuda")[::2]),
        lambda: s2b200.group_norm_act(x, 8, out=x.float()), lambda: s2b200.group_norm_act(x, 8, out_dtype=BF16),
        lambda: s2b200.group_norm_act(x, 8, out=w), lambda: s2b200.group_norm_act(x.t(), 4),
        lambda: s2b200.group_norm_act(x.double(), 8), lambda: s2b200.group_norm_act(grad, 8),
        lambda: s2b200.group_norm_act(x[:1].expand(4, 64).view(4, 1, 64), 8, out=x.view(4, 1, 64)),
        lambda: s2b200.group_norm_act(x.view(1, 4, 64)[:, ::2], 8, out=x.view(1, 4, 64)[:, 1:3]),
        lambda: s2b200.group_norm_act(x, 8, eps=-1.0), lambda: s2b200.group_norm_act(x, 8, err=v),
        lambda: s2b200.linear_act(x, w.float()), lambda: s2b200.linear_act(x, w[:, :32]),
        lambda: s2b200.linear_act(x.float(), w.float()), lambda: s2b200.linear_act(x, w, v),
        lambda: s2b200.linear_act(x, w, activation=None), lambda: s2b200.linear_act(x, w, residual=x),
        lambda: s2b200.linear_act(x, w, out=x), lambda: s2b200.linear_act(x, w, out_dtype=BF16),
        lambda: s2b200.linear_act(x, w.cpu()), lambda: s2b200.linear_act(x, w, residual=x[:, :32].float()),
        lambda: s2b200.linear_act(x, w, out=x[:, :32]), lambda: s2b200.linear_act(grad, w),
        lambda: s2b200.linear_act(x.t(), w.t()), lambda: s2b200.linear_act(x, w, err=v),
    ]
    for i, call in enumerate(calls):
        with pytest.raises(s2b200.S2Error) as e:
            call()
        assert e.value.status in (s2b200.S2_INVALID_ARGUMENT, s2b200.S2_UNSUPPORTED), i
    with torch.no_grad():
        assert torch.equal(s2b200.linear_act(grad, w), s2b200.linear_act(x, w))


def test_err_word_stays_zero():
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    x, w, b, _ = _operands(500, 256, 512, F16, 43, res=False)
    s2b200.linear_act(x, w, b, err=err)
    s2b200.group_norm_act(x.view(5, 100, 512), 32, err=err)
    assert err.item() == 0


# ---- activations -----------------------------------------------------------------------

def _sweep(n):
    """n values over [-12, 12], and the ones where the activations change their form."""
    v = torch.linspace(-12, 12, n, device="cuda")
    v[:8] = torch.tensor([0.0, -0.0, 1e-30, -1e-30, 1e-4, -1e-4, 13.2, -13.3], device="cuda")
    return v


@pytest.mark.parametrize("act", cl.ACTS)
@pytest.mark.parametrize("out_dtype", [F32, F16, BF16], ids=str)
@pytest.mark.parametrize("M,N", [(1, 200001), (20, 20001), (300, 5003)])
def test_activations_of_the_product(M, N, out_dtype, act):
    """0 x 0 + bias: the activation's own error, relative to its result, in the three kernels' epilogues."""
    v = _sweep(N)
    dtype = F16 if out_dtype == F32 else out_dtype
    y = s2b200.linear_act(torch.zeros(M, 8, device="cuda", dtype=dtype), torch.zeros(N, 8, device="cuda", dtype=dtype), v,
                          act, out_dtype=out_dtype)
    want, room = cl.activation_exact(v, act)
    cl.check(y, want.expand(M, N), room.expand(M, N), act)


@pytest.mark.parametrize("act", cl.ACTS)
@pytest.mark.parametrize("out_dtype", [F32, F16, BF16], ids=str)
@pytest.mark.parametrize("P,pad", [(3, 0), (3, 1)])
def test_activations_of_the_norm(P, pad, out_dtype, act):
    """Equal values: the norm is its bias, exactly."""
    v = _sweep(1 << 16)
    x = _padded(torch.full((2, P, 1 << 16), 3.25, device="cuda"), pad)[1]
    y = s2b200.group_norm_act(x, 1024, None, v, activation=act, out_dtype=out_dtype)
    want, room = cl.activation_exact(v, act)
    cl.check(y, want.expand(y.shape), room.expand(y.shape), act)


# Slices whose blocks turn their buffers over many times with few rows in each: one that reads a buffer before
# its copy has landed, or after the next was begun, meets another unit's rows.
@pytest.mark.parametrize("dtype,out_dtype", [(F16, F16), (F32, F32), (F32, BF16)], ids=str)
@pytest.mark.parametrize("shape", [(2000, 80, 128, 8), (260, 160, 512, 32), (24, 20000, 128, 32), (40, 3600, 512, 32)], ids=str)
def test_norm_of_slices_hands_its_buffers_over(shape, dtype, out_dtype):
    S, P, C, G = shape
    x = _features(shape[:3], _gen(51), dtype)
    x += torch.arange(S, device="cuda", dtype=F32).remainder(17).to(dtype)[:, None, None]
    want = s2b200.group_norm_act(x, G, activation="gelu", out_dtype=out_dtype)
    for s in range(0, S, max(1, S // 60)):
        cl.check(want[s:s + 1], *cl.norm_exact(x[s:s + 1], G, None, None, 1e-6, "gelu"), f"sample {s}")
    off = torch.zeros((), dtype=torch.int64, device="cuda")
    for i in range(60):
        off += (s2b200.group_norm_act(x, G, activation="gelu", out_dtype=out_dtype) != want).sum()
    if dtype == out_dtype:
        for i in range(10):
            y = x.clone()
            off += (s2b200.group_norm_act(y, G, activation="gelu", out=y) != want).sum()
    assert off.item() == 0


# ---- values near fp32's range ------------------------------------------------------------

# rows held by a block, a cluster and (on 4 bytes) a grid; slices joined by each block and by one; the ring
RANGE_SHAPES = [(2, 8, 64, 8), (2, 1500, 512, 32), (1, 60000, 130, 10), (40, 3600, 512, 32), (3, 20001, 512, 32),
                (1, 140000, 512, 32), (1, 300000, 64, 8)]


@pytest.mark.parametrize("dtype,out_dtype", [(F32, F32), (BF16, BF16), (F32, F16)], ids=str)
@pytest.mark.parametrize("how", ["outlier", "first", "spread"])
@pytest.mark.parametrize("shape", RANGE_SHAPES, ids=str)
def test_norm_of_squares_that_overflow(shape, how, dtype, out_dtype):
    """A group whose squares add up beyond fp32 is NaN, all of it; the others do not notice."""
    S, P, C, G = shape
    x = _features(shape[:3], _gen(61), dtype)
    y0 = s2b200.group_norm_act(x, G, activation="relu", out_dtype=out_dtype)
    g, k = G - 1, C // G
    if how == "spread":  # n D^2 beyond 3.4e38, each square below
        x[S - 1, :, g * k:(g + 1) * k] *= 4e18 / x[S - 1, :, g * k:(g + 1) * k].abs().max().item()
        x[S - 1, 0, g * k] = -8e18
        x[S - 1, P - 1, g * k] = 8e18
        x[S - 1, P // 2, g * k:(g + 1) * k] = 1.2e19
        x[S - 1, P // 3, g * k:(g + 1) * k] = -1.2e19
    else:
        x[S - 1, 0 if how == "first" else P // 2 + 1, g * k + k // 2] = 1e20
    y = s2b200.group_norm_act(x, G, activation="relu", out_dtype=out_dtype)
    assert torch.isnan(y[S - 1, :, g * k:(g + 1) * k]).all()
    y[S - 1, :, g * k:(g + 1) * k] = y0[S - 1, :, g * k:(g + 1) * k]
    assert torch.equal(y, y0)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
@pytest.mark.parametrize("shape", RANGE_SHAPES, ids=str)
def test_norm_of_large_values_that_do_not(shape, dtype):
    """max(n, 256) D^2 just within fp32: D = 6 spreads at most.

    The mean of these is about 0, but what its joins round are the means m_i of the parts, by 2^-24 |m_i| each and at
    most 24 times: weighted with n_i / n that is at most 24 2^-24 mean |x| <= 24 2^-24 sqrt(m^2 + sigma^2), so 24 2^-24
    of sigma comes on top of norm_exact's room, whose term is 2^-18 |m| alone: in z 24 2^-24 sigma / sigma."""
    S, P, C, G = shape
    x = _normal(shape[:3], _gen(62)).clamp(-5.9, 5.9)
    scale = (3e38 / max(P * C // G, 256)) ** 0.5 / 6
    x = (x * scale).to(dtype)
    y = s2b200.group_norm_act(x, G)
    for s in {0, S - 1}:
        want, room = cl.norm_exact(x[s:s + 1], G, None, None, 1e-6, "none")
        cl.check(y[s:s + 1], want, room + 24 * 2.0 ** -24)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
# the last two: a last part with one row, and lanes without any
@pytest.mark.parametrize("shape", sorted(set(SLICES + RANGE_SHAPES)) + [(1, 20061, 128, 32), (1, 20061, 512, 32)], ids=str)
def test_norm_about_a_huge_mean(shape, dtype):
    """The mean's own square may be beyond fp32: only distances count."""
    S, P, C, G = shape
    b = torch.linspace(-1, 1, C, device="cuda")
    x = torch.full(shape[:3], 1e20, device="cuda", dtype=dtype)
    y = s2b200.group_norm_act(x, G, None, b)
    assert torch.equal(y, b.to(dtype).expand_as(y))


# ---- waits that run out --------------------------------------------------------------------

# blocks that wait for one another: slices joined by each block and by one, rows on 4 bytes on a grid, the ring
WAITING = [((40, 3600, 512, 32), F16, 0), ((3, 20001, 512, 32), F16, 0), ((1, 60000, 130, 10), F32, 1),
           ((1, 140000, 512, 32), BF16, 0)]


@pytest.mark.parametrize("shape,dtype,pad", WAITING, ids=str)
def test_norm_wait_that_runs_out(shape, dtype, pad):
    """A limit of 1 ns that no block can keep: the kernel ends, says so, writes y's rows only, and the next call is
    right."""
    import time
    x = _padded(_features(shape[:3], _gen(71), dtype), pad)[1]
    want = s2b200.group_norm_act(x, shape[3], activation="silu")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    buf, out = _padded(torch.zeros_like(want), 8)
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    s2b200.lib().s2_debug_norm_wait(1)
    s2b200.group_norm_act(x, shape[3], activation="silu", out=out, err=err)
    assert err.item() == 96
    assert time.perf_counter() - t0 < 0.5
    assert torch.isnan(buf[..., shape[2]:]).all()
    err.zero_()
    for _ in range(3):
        assert torch.equal(s2b200.group_norm_act(x, shape[3], activation="silu", err=err), want)
    assert err.item() == 0


def test_waits_that_run_out_without_a_word_are_asked_for():
    """A call without `err`: the device's own word says so once, and only for what ran on it."""
    assert s2b200.operator_device_error() == 0
    shape, dtype, _ = WAITING[1]
    x = _features(shape[:3], _gen(72), dtype)
    want = s2b200.group_norm_act(x, shape[3])
    torch.cuda.synchronize()
    s2b200.lib().s2_debug_norm_wait(1)
    s2b200.group_norm_act(x, shape[3])
    assert s2b200.operator_device_error("cuda:0") == 96
    assert s2b200.operator_device_error() == 0
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    s2b200.lib().s2_debug_norm_wait(1)
    s2b200.group_norm_act(x, shape[3], err=err)
    assert err.item() == 96 and s2b200.operator_device_error() == 0
    assert torch.equal(s2b200.group_norm_act(x, shape[3]), want)
    s2b200.linear_act(x[0, :300, :512], x[1, :512, :512])
    assert s2b200.operator_device_error() == 0


_CAPTURED_FIRST = r"""
import sys
sys.path.insert(0, sys.argv[1])
import torch, s2b200
x = torch.randn(3, 20001, 512, device="cuda").half()
w = torch.randn(512, 512, device="cuda").half()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    y = s2b200.group_norm_act(x, 32, activation="silu")
    z = s2b200.linear_act(y, w)
    v = s2b200.linear_act(y[0, :1], w)
    u = s2b200.linear_act(y[0, :40, :511], w[:, :511])
y.zero_(), z.zero_(), v.zero_(), u.zero_()
g.replay()
torch.cuda.synchronize()
a = s2b200.group_norm_act(x, 32, activation="silu")
assert torch.equal(a, y) and torch.equal(s2b200.linear_act(a, w), z) and torch.equal(s2b200.linear_act(a[0, :1], w), v)
assert torch.equal(s2b200.linear_act(a[0, :40, :511], w[:, :511]), u)
assert s2b200.operator_device_error() == 0
print("done")
"""


def test_first_calls_of_a_process_inside_a_capture():
    import os
    import subprocess
    import sys
    r = subprocess.run([sys.executable, "-c", _CAPTURED_FIRST, os.path.dirname(os.path.dirname(s2b200.__file__))],
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "done" in r.stdout, r.stderr


@pytest.mark.parametrize("shape", [(0, 64), (3, 0, 64), (0, 3, 64), (2, 3, 0, 64), (2, 0, 3, 64)], ids=str)
def test_no_rows_of_any_shape(shape):
    x = torch.empty(shape, device="cuda", dtype=F16)
    w = torch.ones(32, 64, device="cuda", dtype=F16)
    y = s2b200.linear_act(x, w, residual=torch.empty(shape[:-1] + (32,), device="cuda", dtype=F16))
    assert y.shape == shape[:-1] + (32,)
    assert s2b200.linear_act(x, w, out=y) is y
    assert s2b200.group_norm_act(x, 8).shape == shape
    assert s2b200.group_norm_act(x[None], 8, out=torch.empty_like(x[None])).shape == (1,) + shape


@pytest.mark.parametrize("kw", [dict(groups=1 << 40), dict(groups=8.0), dict(groups=8, eps=None), dict(groups=8, eps=1e39),
                                dict(groups=-8), dict(groups=8, eps=float("nan"))], ids=str)
def test_numbers_out_of_range_are_refused_like_others(kw):
    with pytest.raises(s2b200.S2Error) as e:
        s2b200.group_norm_act(torch.zeros(2, 5, 64, device="cuda"), **kw)
    assert e.value.status == s2b200.S2_INVALID_ARGUMENT


@pytest.mark.parametrize("op", ["norm", "linear"])
def test_tensors_let_go_of_before_another_stream_reads_them(op):
    """With `stream`, the call's tensors may be dropped at once, though the stream is busy: what is allocated and written
    next does not take their place."""
    gen = _gen(81)

    def tensors():
        if op == "norm":
            return [_features((3, 20001, 512), gen, F16), 1 + 0.1 * _normal((512,), gen), _normal((512,), gen)]
        x, w, b, r = _operands(3000, 520, 1000, F16, 82)
        return [x, w, b, r]

    def call(t, **kw):
        if op == "norm":
            return s2b200.group_norm_act(t[0], 32, t[1], t[2], activation="silu", **kw)
        return s2b200.linear_act(t[0], t[1], t[2], "silu", t[3], **kw)

    held = tensors()
    want = call(held)
    side = torch.cuda.Stream()
    for _ in range(3):
        dropped = [t.clone() for t in held]
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(100_000_000)
        got = call(dropped, stream=side)
        shapes = [(t.shape, t.dtype) for t in dropped]
        del dropped
        fresh = [torch.full(s, 7.0, dtype=d, device="cuda") for s, d in shapes for _ in range(2)]
        side.synchronize()
        assert torch.equal(got, want)
        del fresh


def test_outputs_that_require_gradients_are_refused():
    x = torch.zeros(4, 64, dtype=F16, device="cuda")
    out = torch.zeros(4, 64, dtype=F16, device="cuda", requires_grad=True)
    for call in (lambda: s2b200.group_norm_act(x, 8, out=out), lambda: s2b200.linear_act(x, torch.zeros_like(x[:1].expand(64, 64)), out=out)):
        with pytest.raises(s2b200.S2Error):
            call()
        with torch.no_grad():
            assert call() is out


@pytest.mark.parametrize("types", NORM_TYPES, ids=lambda t: f"{t[0]}-{t[1]}".replace("torch.", ""))
@pytest.mark.parametrize("shape", [(1, 24000, 32, 8), (1, 22000, 48, 16), (1, 21500, 32, 1), (2, 25001, 40, 5)], ids=str)
def test_norm_of_small_shares_of_narrow_slices(shape, types):
    S, P, C, G = shape
    x = _features(shape[:3], _gen(91), types[0])
    for act in ("silu", "none"):
        y = s2b200.group_norm_act(x, G, activation=act, out_dtype=types[1])
        cl.check(y, *cl.norm_exact(x, G, None, None, 1e-6, act))
    off = torch.zeros((), dtype=torch.int64, device="cuda")
    for _ in range(50):
        off += (s2b200.group_norm_act(x, G, out_dtype=types[1]) != y).sum()
    assert off.item() == 0


def test_captured_on_the_stream_that_is_passed():
    """`stream` may be the one that is being captured; what the calls hand on may be dropped inside the capture."""
    gen = _gen(95)
    x = _features((3, 20001, 512), gen, F16)
    w, b = (_normal((512, 512), gen) * 0.05).half(), _normal((512,), gen)
    side = torch.cuda.Stream()

    def run(**kw):
        h = s2b200.group_norm_act(x, 32, activation="silu", **kw)
        a = s2b200.linear_act(h, w, b, **kw)
        del h
        h = s2b200.linear_act(a, w, b, "gelu", x, **kw)
        del a
        return s2b200.group_norm_act(h, 16, b, **kw)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        y = run(stream=side)
    for seed in (96, 97):
        x.copy_(_features((3, 20001, 512), _gen(seed), F16))
        want = run()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)
    assert s2b200.operator_device_error() == 0
