"""What the 8-bit operators refuse, their plans and their status word: nothing here launches a kernel."""
import pytest
import torch

from crosslayer_transcoder_b200 import fp8
from crosslayer_transcoder_b200._lib import CltError, lib
from crosslayer_transcoder_b200.model import CrosslayerDecoder, CrossLayerTranscoder, Encoder, JumpReLU


def _block(R=256, C=256, rows=128, Z=None):
    lead = () if Z is None else (Z,)
    return fp8.BlockTensor(torch.zeros(*lead, R, C).to(torch.float8_e4m3fn), torch.ones(*lead, -(-R // rows), -(-C // 128)), rows)


@pytest.mark.parametrize("call, error", [
    (lambda: fp8.quantize([1.0]), TypeError),
    (lambda: fp8.quantize(torch.zeros(4, 4, dtype=torch.float64)), TypeError),
    (lambda: fp8.quantize(torch.zeros(4)), ValueError),
    (lambda: fp8.quantize(torch.zeros(1, 1, 4, 4)), ValueError),
    (lambda: fp8.quantize(torch.zeros(4, 4), block_rows=64), ValueError),
    (lambda: fp8.BlockTensor(torch.zeros(4, 4), torch.ones(1, 1)), TypeError),
    (lambda: fp8.BlockTensor(torch.zeros(4, 4).to(torch.float8_e4m3fn), torch.ones(1, 2)), ValueError),
    (lambda: fp8.BlockTensor(torch.zeros(4, 4).to(torch.float8_e4m3fn), torch.ones(4, 1)), ValueError),
    (lambda: fp8.BlockTensor(torch.zeros(4, 4).to(torch.float8_e4m3fn), torch.ones(1, 1).double()), TypeError),
    (lambda: fp8.BlockTensor(torch.zeros(4, 4).to(torch.float8_e4m3fn), torch.ones(1, 1), block_rows=2), ValueError),
    (lambda: _block()[0], ValueError),
    (lambda: _block(Z=2)[0:1], ValueError),
    (lambda: _block().dequantize(torch.float64), ValueError),
    (lambda: fp8.matmul(torch.zeros(4, 4), _block()), TypeError),
    (lambda: fp8.matmul(_block(), _block(Z=1)), ValueError),
    (lambda: fp8.matmul(_block(C=128), _block()), ValueError),
    (lambda: fp8.matmul(_block(Z=2), _block(Z=3)), ValueError),
    (lambda: fp8.matmul(_block(), _block(rows=1)), ValueError),
    (lambda: fp8.matmul(_block(rows=1).mT, _block()), ValueError),
    (lambda: fp8.matmul(_block(), _block(), out_dtype=torch.float64), ValueError),
    (lambda: fp8.matmul(_block(), _block(), bias=torch.zeros(255)), ValueError),
    (lambda: fp8.matmul(_block(), _block(), bias=torch.zeros(256, dtype=torch.int32)), TypeError),
    (lambda: fp8.project(torch.zeros(2, 3, 4), torch.zeros(3, 5, 6)), ValueError),
    (lambda: fp8.project(torch.zeros(2, 2, 4), torch.zeros(3, 4, 6)), ValueError),
    (lambda: fp8.project(torch.zeros(4), torch.zeros(3, 4, 6)), ValueError),
    (lambda: fp8.project(torch.zeros(2, 4), torch.zeros(4)), ValueError),
    (lambda: fp8.project(torch.zeros(2, 0), torch.zeros(0, 3)), ValueError),
    (lambda: fp8.project(torch.zeros(2, 4), torch.zeros(4, 6), torch.zeros(5)), ValueError),
    (lambda: fp8.project(torch.zeros(2, 4).long(), torch.zeros(4, 6)), TypeError),
    (lambda: fp8.crosslayer_decode(torch.zeros(5, 2, 4), [torch.zeros(1, 4, 3)]), ValueError),
    (lambda: fp8.crosslayer_decode(torch.zeros(5, 2, 4), [torch.zeros(1, 4, 3), torch.zeros(1, 4, 3)]), ValueError),
    (lambda: fp8.crosslayer_decode(torch.zeros(5, 2, 4), [torch.zeros(1, 4, 3), torch.zeros(2, 4, 2)]), ValueError),
    (lambda: fp8.crosslayer_decode(torch.zeros(5, 1, 4), [torch.zeros(1, 4, 3)], torch.zeros(3)), ValueError),
    (lambda: fp8.crosslayer_decode(torch.zeros(5, 0, 4), []), ValueError),
    (lambda: fp8.project(torch.zeros(1, 362, 1), torch.zeros(362, 1, 1)), ValueError),
    (lambda: fp8.jump_relu(torch.tensor(1.0)), ValueError),
    (lambda: fp8.jump_relu(torch.zeros(3, 4), torch.zeros(3)), ValueError),
    (lambda: fp8.jump_relu(torch.zeros(4), torch.zeros(2, 4)), ValueError),
    (lambda: fp8.jump_relu(torch.zeros(3, 4), torch.zeros(4), bandwidth=0.0), ValueError),
    (lambda: fp8.jump_relu(torch.zeros(3, 4), torch.zeros(4), bandwidth=float("nan")), ValueError),
    (lambda: fp8.jump_relu(torch.zeros(3, 4), torch.zeros(4), bandwidth=torch.ones(2)), ValueError),
])
def test_refusals(call, error):
    with pytest.raises(error):
        call()


@pytest.mark.parametrize("call", [
    lambda: fp8.quantize(torch.zeros(4, 4)),
    lambda: _block().dequantize(),
    lambda: fp8.matmul(_block(), _block()),
    lambda: fp8.project(torch.zeros(2, 4), torch.zeros(4, 6)),
    lambda: fp8.crosslayer_decode(torch.zeros(5, 1, 4), [torch.zeros(1, 4, 3)]),
    lambda: fp8.jump_relu(torch.zeros(3, 4), torch.zeros(4)),
])
def test_cpu_tensors_are_refused(call):
    with pytest.raises(CltError, match="CUDA"):
        call()


def test_model_switch():
    model = CrossLayerTranscoder(JumpReLU(0.03, 1.0, 2, 24), Encoder(8, 24, 2), CrosslayerDecoder(8, 24, 2))
    x = torch.randn(3, 2, 8)
    before = model(x)
    assert "eight_bit" not in str(model.to_config()) and not model.eight_bit
    model.eight_bit = True
    with pytest.raises(CltError, match="CUDA"):
        model(x)
    model.eight_bit = False
    assert all(torch.equal(a, b) for a, b in zip(before, model(x)))


def test_views():
    b = _block(100, 300, 1, Z=2)
    assert b.shape == (2, 100, 300) and b.mT.shape == (2, 300, 100) and b[1].shape == (100, 300) and b.mT.mT.shape == b.shape
    assert b[0].mT.shape == (300, 100) and "block_rows=1" in repr(b)


@pytest.mark.parametrize("mode, M, N, K, L", [(0, 257, 768, 120000, 1), (0, 1, 768, 24576, 1), (0, 1, 1, 1, 1), (1, 257, 768, 10000, 12),
                                              (2, 5, 10000, 768, 12), (3, 320, 2001, 7, 6), (0, 33, 200, 20000, 3), (1, 64, 64, 64, 361)])
def test_parts_cover_the_contraction(mode, M, N, K, L):
    """Parts are at least two to a slab where there are any, of four blocks or more each, and few enough for a grid."""
    parts = lib().query("clt_fp8_matmul_parts", mode, M, N, K, L, 148)
    slabs = L * (L + 1) // 2 if mode == 3 else L
    chain = {0: 1, 1: L, 2: L, 3: 1}[mode] * -(-K // 128)
    assert parts == 0 or (slabs < parts <= 65535 and parts <= slabs * -(-chain // 4))
    assert lib().query("clt_fp8_matmul_parts", mode, M, N, 0, L, 148) == 0


@pytest.mark.parametrize("Z, R, C", [(1, 1, 1), (3, 136, 64), (12, 4000, 10000), (2, 129, 257)])
def test_copies_have_room(Z, R, C):
    """A copy's buffer holds its values, rows of a multiple of 32, and the scales of its blocks, and not 256 bytes more."""
    need = Z * R * (-(-C // 32) * 32) + 4 * Z * -(-R // 128) * -(-C // 128)
    units = lib().query("clt_fp8_copy_units", Z, R, C)
    assert need <= 256 * units < need + 256
    assert lib().query("clt_fp8_copy_units", Z, 0, C) == 0


def test_status_word(monkeypatch):
    """What a kernel reports reaches the next call, once."""
    word = torch.zeros(1, dtype=torch.int32)
    monkeypatch.setattr(fp8, "_status", word)
    monkeypatch.setattr(fp8, "_status_view", word.numpy())
    assert fp8._status_word() is word
    word[0] = 0x12
    with pytest.raises(CltError, match="0x12.*gave up waiting for an accumulator"):
        fp8._status_word()
    assert fp8._status_word() is word


def test_library_refuses():
    """Arguments that the library itself checks, before any launch."""
    call = lib().call
    p = 4096                                            # an address; nothing is read
    with pytest.raises(CltError, match="blocks of 2 rows"):
        call("clt_fp8_quantize", p, 0, 128, 0, p, 128, p, None, 1, 1, 128, 2, None)
    with pytest.raises(CltError, match="column sums"):
        call("clt_fp8_quantize", p, 0, 128, 0, p, 128, p, p, 1, 1, 128, 1, None)
    with pytest.raises(CltError, match="16-byte aligned"):
        call("clt_fp8_quantize", p, 0, 100, 0, p, 100, p, None, 1, 1, 100, 1, None)
    with pytest.raises(CltError, match="misaligned"):
        call("clt_fp8_quantize", p + 2, 0, 128, 0, p, 128, p, None, 1, 1, 128, 1, None)
    one = torch.tensor([0], dtype=torch.int64)          # a host array with a null address
    for n, text in ((0, "bad dims"), (362, "bad dims"), (1, "null")):
        with pytest.raises(CltError, match=text):
            call("clt_fp8_quantize_blocks", one, n, 0, p, 128, p, 4, 128, None)
    with pytest.raises(CltError, match="16-byte aligned"):
        call("clt_fp8_align", p, 100, 0, p, 100, 1, 1, 100, None)
    with pytest.raises(CltError, match="null"):
        call("clt_fp8_dequantize", None, 128, 0, p, 1, 1, 1, 1, p, 0, 1, 1, 128, None)
    with pytest.raises(CltError, match="output type"):
        call("clt_fp8_dequantize", p, 128, 0, p, 1, 1, 1, 1, p, 3, 1, 1, 128, None)
    args = [0, p, 128, 0, 0, p, 1, 1, 1, 128, p, 128, 0, 0, p, 1, 1, 1, None, 0, p, 0, 128, 0, None, 0, 128, 128, 128, 1, p, None]
    for at, value, text in ((0, 4, "bad mode"), (28, 0, "bad mode"), (29, 0, "bad mode"), (9, 2, "blocks of 2"), (21, 3, "output type"),
                            (22, 127, "distance"), (20, p + 2, "misaligned"), (30, None, "null")):
        bad = list(args)
        bad[at] = value
        with pytest.raises(CltError, match=text):
            call("clt_fp8_matmul", *bad)
    bad = list(args)
    bad[4], bad[9] = 1, 1
    with pytest.raises(CltError, match="transposed operand needs 128"):
        call("clt_fp8_matmul", *bad)
    with pytest.raises(CltError, match="bandwidth"):
        call("clt_jump_relu_fwd", p, 8, p, None, 0.0, p, p, 0, 1, 8, None)
    with pytest.raises(CltError, match="null"):
        call("clt_jump_relu_bwd", p, 8, p, p, None, 1.0, p, None, None, 0, 0, 1, 8, None)
    with pytest.raises(CltError, match="scratch"):
        call("clt_jump_relu_bwd", p, 8, p, p, None, 1.0, p, p, p, 3, 0, 1, 8, None)
    fwd = [0, p, 0, 64, 64, p, None, 0, None, p, p, p, None, 0, 4, 1, 64, 64, p, None]
    for at, value, text in ((1, None, "null"), (5, None, "null"), (9, None, "null"), (0, 1, "null"), (14, 0, "bad dims"), (15, 362, "bad dims"),
                            (10, p + 8, "16-byte")):
        bad = list(fwd)
        bad[at] = value
        with pytest.raises(CltError, match=text):
            call("clt_fp8_pass_fwd", *bad)
    bwd = [0, p, 0, 64, 64, p, p, p, p, 0, p, p, 1 << 20, 4, 1, 64, 64, p, None]
    for at, value, text in ((1, None, "null"), (5, None, "null"), (6, None, "null"), (11, None, "null"), (12, 1, "too small"), (11, p + 4, "misaligned"),
                            (16, 0, "bad dims")):
        bad = list(bwd)
        bad[at] = value
        with pytest.raises(CltError, match=text):
            call("clt_fp8_pass_bwd", *bad)
    with pytest.raises(CltError, match="bad dims"):
        call("clt_sum_chunks", p, p, 0, 1, 8, None)


def _meta(*shape, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype, device="meta")


@pytest.mark.parametrize("n", [2 ** 31 - 255, 2 ** 31, 2 ** 32 + 5])
def test_axes_beyond_32_bits_are_refused(n):
    """The library's sizes are C ints: a larger one would arrive as another number."""
    W, decoder = _meta(1, 1, 8), [_meta(1, 1, 8)]
    for call in (lambda: fp8.quantize(_meta(n, 1)), lambda: fp8.quantize(_meta(2, n)), lambda: fp8.quantize(_meta(n, 1, 1)),
                 lambda: fp8.BlockTensor(_meta(n, 1, dtype=torch.float8_e4m3fn), _meta(n, 1, dtype=torch.float32), 1),
                 lambda: fp8.project(_meta(n, 1, 1), W), lambda: fp8.project(_meta(n // 2 + 1, 2, 1, 1), W),
                 lambda: fp8.project(_meta(4, 1), _meta(1, n)), lambda: fp8.crosslayer_decode(_meta(n, 1, 1), decoder),
                 lambda: fp8.crosslayer_decode(_meta(4, 1, n), [_meta(1, n, 2)]),
                 lambda: fp8.jump_relu(_meta(n)), lambda: fp8.jump_relu(_meta(n, 1), _meta(1))):
        with pytest.raises(ValueError, match="at most"):
            call()


def test_largest_axis_is_taken():
    with pytest.raises(CltError, match="CUDA tensors only"):
        fp8.quantize(_meta(fp8.MOST, 1))


def test_a_stack_is_indexed_with_integers_alone():
    with pytest.raises(ValueError):
        _block(Z=2)[True]
    assert _block(Z=2)[-1].shape == (256, 256)
