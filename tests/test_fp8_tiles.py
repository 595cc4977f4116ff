"""Every cut of an 8-bit product (jl_fp8_cut) against the definition, at a shape that the rule sends there; rows far apart and the greatest depths that tiles take.

Operands are whole numbers times powers of two whose sums stay below 2^23 steps: exact in any order, so linear results are compared for equality.  The reference is a product in 64 bits."""
import ctypes as C

import pytest
import torch

from .test_fp8 import E4, E8, F32, UNIT_SLACK, check, gen, gpu, scales, unit64


def cut(LO, x, w, gated=False):
    """The cut's name and how many shares of the depth."""
    from jacobiforcing_amd import _native as N
    shares = C.c_int32()
    return N.layers().jl_fp8_cut(LO._fp8_operands(x, w, "test"), int(gated), C.byref(shares)).decode(), shares.value


def whole(n, k, o, scale, seed, most, x_ld=None, w_ld=None):
    """(x, w, product in 64 bits), made on the GPU; ``x_ld``, ``w_ld``: rows so many bytes apart."""
    from jacobiforcing_amd import layer_ops as LO
    assert k * most * most * 2 < 2 ** 20                # steps of 2^-3
    g, kb, rb = torch.Generator("cuda").manual_seed(seed), k // 128, -(-o // 128)
    draw = lambda lo, hi, *size: torch.randint(lo, hi, size, generator=g, device="cuda")
    xe, we = torch.zeros(kb, -(-n // 16) * 16, dtype=torch.int64, device="cuda"), draw(-2, 1, rb, kb)
    xe[:, :n] = draw(-1, 2, kb, n)
    held = (lambda e: (e + 127).to(torch.uint8).view(E8)) if scale == E8 else (lambda e: torch.exp2(e.float()))
    room = lambda rows, ld: torch.empty(rows, ld or k, dtype=torch.uint8, device="cuda").view(E4)[:, :k]
    x, w = room(n, x_ld), room(o, w_ld)
    want = torch.zeros(n, o, dtype=torch.float64, device="cuda")
    for c in range(0, k, 8192):
        wide = min(8192, k - c)
        b = slice(c // 128, (c + wide) // 128)
        xc, wc = draw(-most, most + 1, n, wide).float(), draw(-most, most + 1, o, wide).float()
        x[:, c:c + wide], w[:, c:c + wide] = xc.to(E4), wc.to(E4)
        xc = xc.double() * torch.exp2(xe[b, :n].t().double()).repeat_interleave(128, 1)
        wc = wc.double() * torch.exp2(we[:, b].double()).repeat_interleave(128, 1).repeat_interleave(128, 0)[:o]
        want += xc @ wc.t().contiguous()
    return LO.Fp8Rows(x, held(xe)[:, :n].t()), LO.Fp8Weight(w, held(we)), want


def linear(LO, x, w, want, o):
    assert torch.equal(LO.linear_fp8(x, w, None, F32).double(), want)
    bias = torch.randint(-8, 9, (o,), generator=gen(o)).float().cuda()
    assert torch.equal(LO.linear_fp8(x, w, bias), (want + bias.double()).float().bfloat16())


@gpu
@scales
@pytest.mark.parametrize("n,k,o,name,shared", [
    (9, 256, 70000, "16x128 many", False), (24, 256, 70001, "32x128 many", False), (50, 256, 70000, "64x128 many", False), (2, 256, 70000, "rows", False),
    (12, 18944, 512, "16x64", True), (24, 512, 130, "32x64", False), (24, 3584, 130, "32x64", True), (100, 512, 4608, "64x64", False), (40, 9472, 2100, "64x64", True),
    (1100, 512, 1500, "64x128", False), (256, 3584, 4608, "64x128", False), (70, 9472, 2100, "64x128", True), (1030, 512, 2100, "128x128", False), (128, 18944, 3584, "128x128", True),
    (1030, 128, 20000, "128x128 two", False), (1030, 384, 20000, "128x128 two", False), (2050, 512, 2100, "128x256", False), (512, 18944, 3584, "128x256", True), (2050, 512, 4608, "256x256", False),
    (1000, 18944, 3584, "256x256", True), (8200, 640, 5001, "256x256", False)])
def test_products(n, k, o, name, shared, scale):
    from jacobiforcing_amd import layer_ops as LO
    x, w, want = whole(n, k, o, scale, n + k + o, 2 if k > 9000 else 3)
    assert cut(LO, x, w)[0] == name and (cut(LO, x, w)[1] > 1) == shared
    linear(LO, x, w, want, o)


def sixtyfourth(w):
    """w / 64: sums some units large."""
    return w._replace(scale=(w.scale.view(torch.uint8) - 6).view(E8) if w.scale.dtype == E8 else w.scale / 64)


# the last one: 400 tiles, more than one for a workgroup
@gpu
@scales
@pytest.mark.parametrize("n,k,o,name", [(1, 512, 256, "16x256"), (2050, 512, 512, "32x256"), (2050, 512, 1024, "64x256"), (2050, 512, 2048, "128x256"), (2050, 512, 4608, "256x256"), (6200, 1024, 4096, "256x256")])
@pytest.mark.parametrize("kind", [1, 2])
def test_gated_products(n, k, o, name, kind, scale):
    from jacobiforcing_amd import layer_ops as LO
    x, w, z = whole(n, k, o, scale, n + k + o, 3)
    z = z.cpu() / 64
    w, F = sixtyfourth(w), o // 2
    assert cut(LO, x, w, True) == (name, 1) and float(z.abs().max()) < 32
    h, extra = unit64(z[:, :F], z[:, F:], kind, 2.0, 1.5, 0.5)
    check(LO.linear_gated_fp8(x, w, kind, 2.0, 1.5, 0.5), h, scale, UNIT_SLACK, extra)


FAR = 1 << 24                                           # the farthest that tiles take


@gpu
@scales
@pytest.mark.parametrize("n,k,o,x_ld,w_ld,tiles", [(600, 256, 520, FAR, FAR, True), (600, 256, 520, FAR + 16, FAR, False), (600, 256, 520, FAR, FAR + 16, False), (2050, 512, 4608, FAR, None, True),
                                                   (8200, 640, 5001, 1 << 20, 1 << 20, True), (40, 256, 300, FAR, FAR, True)])
def test_rows_far_apart(n, k, o, x_ld, w_ld, tiles, scale):
    """Tiles whose first row lies beyond 2^32 bytes and whose last one lies almost 2^32 behind that; 256 rows of x, then as many of w."""
    from jacobiforcing_amd import layer_ops as LO
    x, w, want = whole(n, k, o, scale, n + k + o, 3, x_ld, w_ld)
    assert (cut(LO, x, w)[0] != "rows") == tiles
    linear(LO, x, w, want, o)


@gpu
@scales
@pytest.mark.parametrize("n,k,o,x_ld,w_ld,name", [(2050, 512, 1024, FAR, FAR, "64x256"), (2050, 512, 4608, FAR, None, "256x256"), (300, 512, 512, FAR + 16, FAR, "rows"), (5, 512, 512, FAR + 16, FAR, "rows")])
def test_gated_rows_far_apart(n, k, o, x_ld, w_ld, name, scale):
    from jacobiforcing_amd import layer_ops as LO
    x, w, z = whole(n, k, o, scale, n + k + o, 3, x_ld, w_ld)
    z = z.cpu() / 64
    w, F = sixtyfourth(w), o // 2
    assert cut(LO, x, w, True)[0] == name and float(z.abs().max()) < 32
    h, extra = unit64(z[:, :F], z[:, F:], 2)
    check(LO.linear_gated_fp8(x, w, 2), h, scale, UNIT_SLACK, extra)


# 1024 blocks: as many scales of w as a tile has room for; 1025 go straight from memory
@gpu
@scales
@pytest.mark.parametrize("n,k,o,name", [(4096, 131072, 4096, "256x256"), (300, 131072, 200, "64x128"), (12, 131072, 512, "16x64"), (300, 131200, 200, "rows"), (5, 131200, 200, "rows"), (1, 131072, 200, "16x64")])
def test_depths(n, k, o, name, scale):
    from jacobiforcing_amd import layer_ops as LO
    x, w, want = whole(n, k, o, scale, n + o, 1)
    assert cut(LO, x, w)[0] == name
    linear(LO, x, w, want, o)


@gpu
@scales
@pytest.mark.parametrize("n,k,o,name", [(5, 131072, 512, "16x256"), (300, 131072, 256, "16x256"), (20, 131200, 256, "rows"), (5, 131200, 256, "rows")])
def test_gated_depths(n, k, o, name, scale):
    from jacobiforcing_amd import layer_ops as LO
    x, w, z = whole(n, k, o, scale, n + o, 1)
    z = z.cpu() / 64
    w, F = sixtyfourth(w), o // 2
    assert cut(LO, x, w, True) == (name, 1) and float(z.abs().max()) < 32
    h, extra = unit64(z[:, :F], z[:, F:], 2)
    check(LO.linear_gated_fp8(x, w, 2), h, scale, UNIT_SLACK, extra)


def test_what_tiles_take():
    """The rule's borders, without a GPU: rows 2^24 bytes apart, 1024 blocks, scales of x in whole words."""
    from jacobiforcing_amd import _native as N
    L, shares = N.layers(), C.c_int32()
    ok = dict(x=4096, x_scale=4096, w=4096, w_scale=4097, N=300, x_ld=FAR, x_scale_ld=304, w_ld=FAR, w_scale_ld=1024, K=131072, O=512, scale_type=0)
    tiles = lambda gated, **change: L.jl_fp8_cut(C.byref(N.Fp8Product(**{**ok, **change})), gated, C.byref(shares)) != b"rows"
    for gated in (0, 1):
        assert tiles(gated) and tiles(gated, x_scale=4098, scale_type=1)
        for change in (dict(x_ld=FAR + 16), dict(w_ld=FAR + 16), dict(K=131200), dict(x_scale=4098), dict(x_scale_ld=306)):
            assert not tiles(gated, **change), change
            assert shares.value == 1
    assert L.jl_fp8_cut(None, 0, None) == b"rows"


@gpu
def test_tiles_that_follow_one_another_in_a_graph():
    """256 x 256, more tiles than workgroups, captured and replayed beside eager calls on another stream."""
    from jacobiforcing_amd import layer_ops as LO
    x, wp, _ = whole(6200, 1024, 4097, E8, 1, 3)
    _, wg, _ = whole(6200, 1024, 4096, E8, 2, 3)
    wg = sixtyfourth(wg)
    assert cut(LO, x, wp)[0] == cut(LO, x, wg, True)[0] == "256x256"
    both = lambda x: (LO.linear_fp8(x, wp, None, F32), *LO.linear_gated_fp8(x, wg, 2))
    both(x)
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        out = both(x)
    for i in range(4):
        new = whole(6200, 1024, 300, E8, 10 + i, 3)[0]
        eager = both(new)
        x.data.view(torch.uint8).copy_(new.data.view(torch.uint8))
        x.scale.view(torch.uint8).copy_(new.scale.view(torch.uint8))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            beside = both(new)
        graph.replay()
        torch.cuda.synchronize()
        for a, b, c in zip(out, eager, beside):         # (scales' rows lie across: compared as floats)
            assert torch.equal(a.float(), b.float()) and torch.equal(a.float(), c.float()), i
