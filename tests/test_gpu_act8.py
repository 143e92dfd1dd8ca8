"""8-bit checkpoints on the GPU: bit for bit the torch operations on the host,
within the format's error of the original, at every size and alignment."""

import pytest
import torch

from test1_amd import _native, act8
from test1_amd.act8 import act8_bytes, pack_act8, unpack_act8

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]
SIZES = [1, 15, 16, 17, 127, 128, 129, 2047, 4096 + 8, 100_003]


def values(n, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + n)
    x = torch.randn(n, generator=g) * torch.exp(3 * torch.randn(n // 128 + 1, generator=g)).repeat_interleave(128)[:n]
    x[torch.rand(n, generator=g) < 0.01] *= 50
    return x.clamp(-6e4, 6e4).to(dtype)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", SIZES)
def test_bits_equal_the_host_form(dev, n, dtype, fmt):
    x = values(n, dtype)
    want = pack_act8(x, fmt)
    got = pack_act8(x.to(dev), fmt)
    assert got.numel() == act8_bytes(n) and torch.equal(got.cpu(), want)
    back = unpack_act8(got, (n,), dtype, fmt)
    assert torch.equal(back.cpu(), unpack_act8(want, (n,), dtype, fmt))


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", TYPES)
def test_error_of_the_format(dev, dtype, fmt):
    n = 128 * 301
    x = values(n, dtype, 5)
    # restored in float32, so that no rounding to the type hides the codes' own
    back = unpack_act8(pack_act8(x.to(dev), fmt), (n,), torch.float32, fmt).cpu().double()
    x = x.double()
    most = x.view(-1, 128).abs().amax(1, keepdim=True).expand(-1, 128).reshape(-1)
    # half a step of the code, two roundings of x T / a, one of a / T, one of the product
    half = most / 254 if fmt == "int8" else torch.maximum(x.abs() / 16, most / 448 * 2.0 ** -10)
    assert ((back - x).abs() <= half * (1 + 2.0 ** -20) + most * 2.0 ** -22).all()


@pytest.mark.parametrize("off", range(1, 8))
@pytest.mark.parametrize("dtype", TYPES)
def test_any_element_boundary(dev, off, dtype):
    x = values(1000, dtype).to(dev)
    view = x[off:off + 777]
    got = pack_act8(view)
    assert torch.equal(got, pack_act8(view.clone()))
    buf = torch.full((800,), 7.0, dtype=dtype, device=dev)
    unpack_act8(got, (777,), dtype, out=buf[off:off + 777])
    assert torch.equal(buf[off:off + 777], unpack_act8(got, (777,), dtype))
    assert (buf[:off] == 7).all() and (buf[off + 777:] == 7).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", TYPES)
def test_a_block_that_is_not_finite_comes_back_as_nan(dev, dtype, fmt, bad):
    x = values(400, dtype)
    x[130] = bad
    back = unpack_act8(pack_act8(x.to(dev), fmt), (400,), dtype, fmt).cpu()
    assert back[128:256].isnan().all()
    assert back[:128].isfinite().all() and back[256:].isfinite().all()


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_extremes(dev, fmt):
    """Zeros stay zeros; the smallest and largest magnitudes of a type come back finite."""
    for dtype in TYPES:
        top = torch.finfo(dtype).max
        for v in (0.0, torch.finfo(dtype).tiny, torch.finfo(dtype).smallest_normal / 4, top, -top):
            x = torch.full((130,), v, dtype=dtype)
            x[1::3] = 0.0
            back = unpack_act8(pack_act8(x.to(dev), fmt), (130,), dtype, fmt).cpu()
            assert back.isfinite().all() and (back[1::3] == 0).all()
            assert torch.equal(back, unpack_act8(pack_act8(x, fmt), (130,), dtype, fmt))


def test_every_fp8_code_and_every_bf16_value(dev):
    """All 256 codes restored, all finite 16-bit patterns packed, as on the host."""
    nblocks = 2
    packed = torch.zeros(act8_bytes(256), dtype=torch.uint8)
    packed[:256] = torch.arange(256).to(torch.uint8)
    packed[256:] = torch.ones(nblocks).view(torch.uint8)
    for fmt in ("int8", "fp8"):
        got = unpack_act8(packed.to(dev), (256,), torch.float32, fmt).cpu()
        want = unpack_act8(packed, (256,), torch.float32, fmt)
        assert torch.equal(got[~want.isnan()], want[~want.isnan()]) and torch.equal(got.isnan(), want.isnan())
        bits = torch.arange(65536, dtype=torch.int32).to(torch.int16)
        for dtype in (torch.bfloat16, torch.float16):
            x = bits.view(dtype)
            x = x[x.isfinite()]
            assert torch.equal(pack_act8(x.to(dev), fmt).cpu(), pack_act8(x, fmt))


def test_strides_streams_and_empty(dev):
    x = values(64 * 200, torch.bfloat16).view(64, 200).to(dev)
    assert torch.equal(pack_act8(x.t()), pack_act8(x.t().contiguous()))
    assert torch.equal(pack_act8(x[:, 3:77]), pack_act8(x[:, 3:77].contiguous()))
    assert pack_act8(x[:0]).numel() == 0 and unpack_act8(pack_act8(x[:0]), (0, 200)).shape == (0, 200)
    s = torch.cuda.Stream(device=dev)
    s.wait_stream(torch.cuda.current_stream())
    got = pack_act8(x.t(), stream=s)
    back = unpack_act8(got, (200, 64), stream=s)
    s.synchronize()
    assert torch.equal(got, pack_act8(x.t())) and torch.equal(back, unpack_act8(got, (200, 64)))


def test_replays_of_a_captured_call(dev):
    x = values(5000, torch.bfloat16).to(dev)
    packed = torch.empty(act8_bytes(5000), dtype=torch.uint8, device=dev)
    back = torch.empty_like(x)
    pack_act8(x, out=packed)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pack_act8(x, out=packed)
        unpack_act8(packed, x.shape, x.dtype, out=back)
    for k in range(3):
        x.copy_(values(5000, torch.bfloat16, 100 + k))
        torch.cuda.synchronize()
        graph.replay()
        assert torch.equal(packed, pack_act8(x)) and torch.equal(back, unpack_act8(packed, x.shape))


def test_entry_points_refuse(dev):
    hip = _native.hip()
    x = torch.zeros(256, dtype=torch.bfloat16, device=dev)
    p = torch.zeros(act8_bytes(256) + 16, dtype=torch.uint8, device=dev)
    bf = _native.SF_DTYPE_BF16
    assert hip.sf_act8_pack(x.data_ptr(), bf, 256, p.data_ptr() + 1, 0, None) == 9007
    assert hip.sf_act8_pack(x.data_ptr(), 7, 256, p.data_ptr(), 0, None) == 9003
    assert hip.sf_act8_pack(x.data_ptr(), bf, 256, p.data_ptr(), 2, None) == 9001
    assert hip.sf_act8_unpack(p.data_ptr(), 0, 256, x.data_ptr() + 1, bf, None) == 9001
    assert hip.sf_act8_pack(x.data_ptr(), bf, 256, x.data_ptr(), 0, None) == 9005
    assert act8._LEAST == 2.0 ** -100


@pytest.mark.parametrize("off", [1, 2, 4, 8, 15])
@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_packed_elements_on_any_byte(dev, fmt, off):
    x = values(1000, torch.bfloat16).to(dev)
    want = pack_act8(x, fmt)
    back = unpack_act8(want, (1000,), torch.bfloat16, fmt)
    room = torch.full((act8_bytes(1000) + 32,), 7, dtype=torch.uint8, device=dev)
    at = room[off:off + act8_bytes(1000)]
    assert pack_act8(x, fmt, out=at) is at and torch.equal(at, want)
    assert (room[:off] == 7).all() and (room[off + act8_bytes(1000):] == 7).all()
    assert torch.equal(unpack_act8(at, (1000,), torch.bfloat16, fmt), back)
    out = torch.empty_like(x)
    assert unpack_act8(at, (1000,), torch.bfloat16, fmt, out=out) is out and torch.equal(out, back)
    at.zero_()
    s = torch.cuda.Stream(device=dev)
    s.wait_stream(torch.cuda.current_stream())
    pack_act8(x, fmt, out=at, stream=s)
    got = unpack_act8(at, (1000,), torch.bfloat16, fmt, stream=s)
    s.synchronize()
    assert torch.equal(at, want) and torch.equal(got, back)
