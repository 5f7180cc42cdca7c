"""Refusals of the 8-bit linears and of the log probabilities, before anything reaches a device."""
import ctypes
import os

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from flint_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built")
    return _lib.load()


P = ctypes.c_void_p(256)
ODD = ctypes.c_void_p(264)  # not on 16 bytes


@pytest.mark.parametrize("rows,k", [(0, 64), (-1, 64), (1, 0), (1, 8), (1, 24), (1, 65552), ((1 << 23) + 1, 64)])
def test_shapes_that_8_bit_rows_do_not_take(lib, rows, k):
    need = ctypes.c_int64()
    assert lib.fl_quantize_int8(P, P, P, rows, k, None) == -1
    for m, n in ((rows, 64), (64, rows)) if rows != 1 else ((1, 64),):
        assert lib.fl_gemm_int8_workspace(m, n, k, ctypes.byref(need)) == -1
        assert lib.fl_linear_int8_workspace(m, n, k, ctypes.byref(need)) == -1
        assert lib.fl_gemm_int8(P, P, P, P, P, 0, P, m, n, k, None) == -1
        assert lib.fl_linear_int8(P, P, P, P, 0, P, m, n, k, None) == -1
        assert lib.fl_head_logprobs_workspace(m, n, k, 0, ctypes.byref(need)) == -1
        assert lib.fl_head_logprobs(P, P, P, None, 0, None, P, None, None, None, P, m, n, k, None) == -1


def test_pointers_that_8_bit_rows_do_not_take(lib):
    for i in range(3):
        a = [P, P, P]
        a[i] = None
        assert lib.fl_quantize_int8(*a, 4, 64, None) == -1
    assert lib.fl_quantize_int8(ODD, P, P, 4, 64, None) == -1
    assert lib.fl_quantize_int8(P, ODD, P, 4, 64, None) == -1
    for bad in (None, ODD):
        for i in (0, 2, 4):
            a = [P, P, P, P, P, 0, P]
            a[i] = bad
            assert lib.fl_gemm_int8(*a, 4, 64, 64, None) == -1
        for i in (0, 1, 3, 5):
            a = [P, P, P, P, 0, P]
            a[i] = bad
            assert lib.fl_linear_int8(*a, 400, 64, 64, None) == -1
    for i in (1, 3):
        a = [P, P, P, P, P, 0, P]
        a[i] = None
        assert lib.fl_gemm_int8(*a, 4, 64, 64, None) == -1
    assert lib.fl_gemm_int8_workspace(4, 64, 64, None) == -1
    assert lib.fl_linear_int8_workspace(4, 64, 64, None) == -1


def test_log_probabilities_that_are_refused(lib):
    need = ctypes.c_int64()

    def call(logits=P, stride=1000, rows=4, vocab=1000, tokens=P, top=5, outs=(P, P, P, P, P), work=P):
        return lib.fl_logprobs(logits, 0, stride, rows, vocab, tokens, top, *outs, work, None)

    for rows, vocab, top in ((0, 1000, 5), (4, 0, 0), (4, 1000, 33), (4, 1000, -1), (4, 7, 8), (4, (1 << 20) + 1, 5),
                             ((1 << 17) + 1, 1000, 5)):
        assert call(rows=rows, vocab=vocab, top=top, stride=1 << 21) == -1
        assert lib.fl_logprobs_workspace(rows, vocab, top, ctypes.byref(need)) == -1
    assert call(logits=None) == -1
    assert call(stride=999) == -1                      # rows that overlap
    assert call(outs=(None, P, P, P, P)) == -1         # tokens without a place for their log probabilities
    assert call(outs=(P, None, P, P, P)) == -1
    assert call(outs=(P, P, None, P, P)) == -1
    assert call(outs=(P, P, P, None, P)) == -1
    assert call(outs=(P, P, P, P, None)) == -1
    assert lib.fl_logprobs_workspace(1, 49152, 5, ctypes.byref(need)) == 0 and need.value > 0
    assert call(rows=1, vocab=49152, work=None) == -1  # several chunks of a row need it
    assert call(rows=1, vocab=49152, work=ODD) == -1
    assert lib.fl_head_logprobs_workspace(4, 1000, 64, 33, ctypes.byref(need)) == -1
    for bad in (None, ODD):
        for i in (0, 1, 10):
            a = [P, P, P, P, 5, P, P, P, P, P, P]
            a[i] = bad
            assert lib.fl_head_logprobs(*a, 4, 1000, 64, None) == -1


def test_a_prompt_with_features_needs_its_arguments(lib):
    assert lib.fl_prefill_feat(None, None, P, 4, 0, None, P, P, None) == -1
    assert lib.fl_prefill_feat(None, None, P, 4, 0, None, None, P, None) == -1
    assert lib.fl_prefill_feat(None, None, P, 4, 0, None, ODD, P, None) == -1


def test_host_layer_refuses():
    from flint_amd import generate, quantize
    w, s = torch.zeros(8, 32, dtype=torch.int8), torch.zeros(8)
    x = torch.zeros(2, 32, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        quantize.quantize_int8(x)                      # not on a device
    with pytest.raises(ValueError):
        quantize.linear_int8(x, w, s)
    with pytest.raises(ValueError):
        quantize.gemm_int8(w, s, w, s)
    with pytest.raises(ValueError):
        quantize.gemm_int8(w, s, w, s, out_dtype=torch.float16)
    with pytest.raises(ValueError):
        generate.logprobs(torch.zeros(3, 10))
    with pytest.raises(ValueError):
        generate.head_logprobs(x, w, s)
    with pytest.raises(ValueError):
        quantize.DynamicInt8Linear(40, 8)              # K not a multiple of 16
    with pytest.raises(ValueError):
        quantize.DynamicInt8Linear(32, 8, bias=True)


class _OnDevice(torch.Tensor):
    """A CPU tensor that says it is a device's, so that the host layer runs up to the C call."""
    is_cuda, off16 = True, False

    def data_ptr(self):
        return super().data_ptr() + (4 if self.off16 else 0)


def _device_tensor(t, off16=False):
    t = t.as_subclass(_OnDevice)
    t.off16 = off16
    return t


@pytest.fixture
def c_calls(monkeypatch):
    """The host layer without a device: C calls end in a list of (name, whether each of the copies made for it on 16
    bytes was still held when it was made)."""
    import contextlib
    import gc
    import weakref
    from flint_amd import _lib, generate, quantize
    copies, calls = [], []
    real = quantize.aligned16

    def copying(t):
        c = real(t)
        if c is not t:
            copies.append(weakref.ref(c))
        return c

    def call(name, *args):
        if "workspace" in name:
            return 0
        gc.collect()
        calls.append((name, [c() is not None for c in copies]))
        return 0

    monkeypatch.setattr(quantize, "aligned16", copying)
    monkeypatch.setattr(quantize, "_int8_fast", None)
    monkeypatch.setattr(generate, "_head_logprobs_fast", None)
    monkeypatch.setattr(_lib, "call", call)
    monkeypatch.setattr(_lib, "stream_ptr", lambda stream=None: None)
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    return calls


def test_copies_on_16_bytes_live_until_the_launch(c_calls):
    """A copy that is freed before the launch can be given to the next one, which then overwrites what the kernel reads:
    two operands of one size that both start off 16 bytes."""
    from flint_amd import generate, quantize
    w, s = _device_tensor(torch.zeros(8, 32, dtype=torch.int8), True), _device_tensor(torch.zeros(8))
    xq = _device_tensor(torch.zeros(8, 32, dtype=torch.int8), True)
    x = _device_tensor(torch.zeros(8, 32, dtype=torch.bfloat16), True)
    quantize.gemm_int8(xq, s, w, s)
    quantize.quantize_int8(x, _device_tensor(torch.zeros(8, 32, dtype=torch.int8)), s)
    quantize.linear_int8(x, w, s)
    generate.head_logprobs(x, w, s)
    assert [n for n, _ in c_calls] == ["fl_gemm_int8", "fl_quantize_int8", "fl_linear_int8", "fl_head_logprobs"]
    made = 0
    for (name, held), n in zip(c_calls, (2, 1, 1, 1)):  # linear_int8's and head_logprobs' rows lose the mark on their way
        assert held[made:] == [True] * n, name
        made += n


def test_the_scale_is_the_product():
    """At every bf16 significand: s = fp32(max fp32(1 / 127)), computed here in whole numbers; where that is an ulp below
    fp32(max / 127), half the maximum is 64, and 63.5 steps to even, 64, elsewhere or 63."""
    from fractions import Fraction
    from oracle import scoring

    def fp32(x):  # of a positive fraction, to nearest even
        e = 0
        while x >= 1 << 24:
            x, e = x / 2, e + 1
        while x < 1 << 23:
            x, e = x * 2, e - 1
        return Fraction(round(x)) * Fraction(2) ** e

    rec, below = fp32(Fraction(1, 127)), []
    for top in range(128, 256):
        x = torch.tensor([[top, top / 2, -top / 2] + [0.0] * 13]).to(torch.bfloat16)
        q, s = scoring.quantize_rows(x)
        product, quotient = fp32(top * rec), fp32(Fraction(top, 127))
        assert Fraction(float(s[0])) == product
        half = round(Fraction(top, 2) / product)  # ties to even
        assert q[0, :3].tolist() == [127, half, -half]
        if product != quotient:
            below.append(top)
            assert product < quotient and half == 64 and round(Fraction(top, 2) / quotient) == 63
        else:
            assert half in (63, 64)
    assert below == [143, 144, 175, 207, 208, 239]


@pytest.mark.parametrize("cast", [lambda m: m.to(torch.bfloat16), lambda m: m.bfloat16(), lambda m: m.half(),
                                  lambda m: m.to("meta", torch.bfloat16), lambda m: m.double(),
                                  lambda m: torch.nn.Sequential(m).to(device="cpu", dtype=torch.bfloat16)[0]])
def test_scales_stay_fp32_when_the_model_is_cast(cast):
    """A model is put into its precision as a whole; the scales are no activations' type."""
    from flint_amd.quantize import DynamicInt8Linear
    m = DynamicInt8Linear(32, 8)
    m.scales.copy_(torch.arange(8) + 1 / 3)
    m.weight.fill_(5)
    scales = m.scales.clone()
    m = cast(m)
    assert m.scales.dtype == torch.float32 and m.weight.dtype == torch.int8
    assert m.scales.device == m.weight.device and "scales" in m.state_dict()
    assert m.scales.is_meta or torch.equal(m.scales, scales)
