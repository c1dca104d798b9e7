"""What the microscaled 4-bit entry points and the sampler refuse, before any work reaches the device (run
without one)."""
import ctypes as C
import os
import re

import pytest

from helpers import ROOT, twd

P = 1 << 20  # an aligned address that no refused call reads


def refused(rc, code, words):
    t = twd()
    assert rc == code
    assert words in t.last_error()


def test_library_exports_what_the_headers_declare():
    t = twd()
    for name, count in (("twd_mx.h", 7), ("twd_sampler.h", 3)):
        text = open(os.path.join(ROOT, "include", name)).read()
        syms = re.findall(r"TWD_API\s+[\w\s\*]+?\b(twd_\w+)\s*\(", text)
        assert len(syms) == count and all(hasattr(t.lib, s) for s in syms)


def test_quantize_refusals():
    t = twd()
    q = t.lib.twd_mx_quantize
    inv = t.TWD_E_INVALID
    refused(q(None, 0, 1, 32, 32, P, P, None), inv, "null")
    refused(q(P, 0, 1, 32, 32, None, P, None), inv, "null")
    refused(q(P, 0, 1, 32, 32, P, None, None), inv, "null")
    refused(q(P, 3, 1, 32, 32, P, P, None), inv, "type")
    refused(q(P, 0, 0, 32, 32, P, P, None), inv, "no rows")
    refused(q(P, 0, 1, 0, 32, P, P, None), inv, "multiple of 32")
    refused(q(P, 0, 1, 48, 48, P, P, None), inv, "multiple of 32")
    refused(q(P, 0, 2, 64, 63, P, P, None), inv, "stride")
    refused(q(P + 2, 0, 1, 32, 32, P, P, None), inv, "aligned")
    refused(q(P + 1, 1, 1, 32, 32, P, P, None), inv, "aligned")
    refused(q(P, 0, 1, 32, 32, P + 4, P, None), inv, "16 bytes")


def test_dequantize_refusals():
    t = twd()
    q = t.lib.twd_mx_dequantize
    inv = t.TWD_E_INVALID
    refused(q(None, P, 1, 32, P, 0, 32, None), inv, "null")
    refused(q(P, None, 1, 32, P, 0, 32, None), inv, "null")
    refused(q(P, P, 1, 32, None, 0, 32, None), inv, "null")
    refused(q(P, P, 1, 32, P, -1, 32, None), inv, "type")
    refused(q(P, P, 0, 32, P, 0, 32, None), inv, "no rows")
    refused(q(P, P, 1, 33, P, 0, 33, None), inv, "multiple of 32")
    refused(q(P, P, 2, 64, P, 0, 32, None), inv, "stride")
    refused(q(P, P, 1, 32, P + 1, 2, 32, None), inv, "aligned")
    refused(q(P + 8, P, 1, 32, P, 0, 32, None), inv, "16 bytes")


def test_head_refusals():
    t = twd()
    inv = t.TWD_E_INVALID
    h = C.c_void_p()
    create = t.lib.twd_mxhead_create
    refused(create(P, P, 16, 32, 0.0, None, None), inv, "null")
    refused(create(None, P, 16, 32, 0.0, None, C.byref(h)), inv, "null")
    refused(create(P, None, 16, 32, 0.0, None, C.byref(h)), inv, "null")
    refused(create(P, P, 0, 32, 0.0, None, C.byref(h)), inv, "vocab")
    refused(create(P, P, (1 << 30) + 1, 32, 0.0, None, C.byref(h)), inv, "vocab")
    for d in (0, 16, 40, (1 << 20) + 32):
        refused(create(P, P, 16, d, 0.0, None, C.byref(h)), inv, "d_model")
    for cap in (-1.0, float("nan"), float("inf"), 1e-31, 1e31):
        refused(create(P, P, 16, 32, cap, None, C.byref(h)), inv, "softcap")
    refused(create(P + 8, P, 16, 32, 0.0, None, C.byref(h)), inv, "16 bytes")
    assert not h
    refused(t.lib.twd_mxhead_logits(None, P, 1, 32, P, 0, 16, None), inv, "null head")
    refused(t.lib.twd_mxhead_logits_mx(None, P, P, 1, P, 0, 16, None), inv, "null head")
    refused(t.lib.twd_mxhead_info(None, None, None, None, None), inv, "null head")
    t.lib.twd_mxhead_destroy(None)


def test_sampler_refusals():
    t = twd()
    inv = t.TWD_E_INVALID
    h = C.c_void_p()
    create = t.lib.twd_sampler_create
    refused(create(100, 1, None), inv, "null")
    for v in (0, 524289):
        refused(create(v, 1, C.byref(h)), inv, "max_vocab")
    for r in (0, 4097):
        refused(create(100, r, C.byref(h)), inv, "max_rows")
    assert not h
    refused(t.lib.twd_sampler_sample(None, P, 0, 10, 1, 10, None, None, None, None, P, P, None, None, None), inv,
            "null sampler")
    t.lib.twd_sampler_destroy(None)


def test_python_refuses_what_is_not_on_a_device_or_not_of_its_shape():
    import torch
    t = twd()
    with pytest.raises(ValueError, match="device tensors"):
        t.mx_quantize(torch.zeros(2, 32))
    with pytest.raises(ValueError, match="float32"):
        t.mx_quantize(torch.zeros(2, 32, dtype=torch.float64))
    with pytest.raises(ValueError, match="adjacent"):
        t.mx_quantize(torch.zeros(32, 64).t())
    with pytest.raises(ValueError, match="two-dimensional"):
        t.mx_quantize(torch.zeros(32))
    with pytest.raises(ValueError, match="scales"):
        t.mx_dequantize(torch.zeros(2, 32, dtype=torch.uint8), torch.zeros(2, 3, dtype=torch.uint8))
    with pytest.raises(ValueError, match="codes"):
        t.MxHead(torch.zeros(2, 32), torch.zeros(2, 2, dtype=torch.uint8))


@pytest.mark.gpu
def test_refusals_of_live_objects():
    import torch
    t = twd()
    inv = t.TWD_E_INVALID
    codes = torch.zeros(20, 32, dtype=torch.uint8, device="cuda:0")
    scales = torch.full((20, 2), 127, dtype=torch.uint8, device="cuda:0")
    head = t.MxHead(codes, scales)
    hh = head.handle
    lg, lmx = t.lib.twd_mxhead_logits, t.lib.twd_mxhead_logits_mx
    refused(lg(hh, None, 1, 64, P, 0, 20, None), inv, "null")
    refused(lg(hh, P, 1, 64, None, 0, 20, None), inv, "null")
    for rows in (0, 65537):
        refused(lg(hh, P, rows, 64, P, 0, 20, None), inv, "rows")
    refused(lg(hh, P, 1, 64, P, 2, 20, None), inv, "fp32 or bf16")
    refused(lg(hh, P, 1, 64, P, 0, 19, None), inv, "stride")
    refused(lg(hh, P + 8, 1, 64, P, 0, 20, None), inv, "16 bytes")
    refused(lg(hh, P, 1, 64, P + 2, 0, 20, None), inv, "aligned")
    refused(lg(hh, P, 2, 63, P, 0, 20, None), inv, "hidden rows' stride")
    refused(lg(hh, P, 2, 68, P, 0, 20, None), inv, "hidden rows' stride")
    refused(lg(hh, P, 2, (1 << 26) + 8, P, 0, 20, None), inv, "hidden rows' stride")
    refused(lmx(hh, P, None, 1, P, 0, 20, None), inv, "null")
    with pytest.raises(ValueError, match="hidden"):
        head.logits(torch.zeros(1, 96, dtype=torch.bfloat16, device="cuda:0"))
    with pytest.raises(ValueError, match="hidden"):
        head.logits(torch.zeros(1, 64, dtype=torch.float16, device="cuda:0"))
    with pytest.raises(ValueError, match="out"):
        head.logits(torch.zeros(1, 64, dtype=torch.bfloat16, device="cuda:0"), out=torch.zeros(1, 21, device="cuda:0"))
    head.close()
    sam = t.Sampler(100, 4)
    f = t.lib.twd_sampler_sample
    none = [None] * 4
    refused(f(sam.handle, None, 0, 10, 1, 10, *none, P, P, None, None, None), inv, "null")
    refused(f(sam.handle, P, 0, 10, 1, 10, *none, None, P, None, None, None), inv, "null")
    refused(f(sam.handle, P, 0, 10, 1, 10, *none, P, None, None, None, None), inv, "null")
    refused(f(sam.handle, P, 5, 10, 1, 10, *none, P, P, None, None, None), inv, "type")
    for v in (0, 101):
        refused(f(sam.handle, P, 0, v, 1, 200, *none, P, P, None, None, None), inv, "vocab")
    for r in (0, 5):
        refused(f(sam.handle, P, 0, 10, r, 10, *none, P, P, None, None, None), inv, "rows")
    refused(f(sam.handle, P, 0, 10, 2, 9, *none, P, P, None, None, None), inv, "stride")
    refused(f(sam.handle, P + 2, 0, 10, 1, 10, *none, P, P, None, None, None), inv, "aligned")
    z = torch.zeros(2, 50, device="cuda:0")
    with pytest.raises(ValueError, match="uniform"):
        sam.sample(z, torch.zeros(3, device="cuda:0"))
    with pytest.raises(ValueError, match="top_k"):
        sam.sample(z, torch.zeros(2, device="cuda:0"), top_k=torch.zeros(2, device="cuda:0"))
    with pytest.raises(ValueError, match="one call"):
        sam.sample(z, torch.zeros(2))
    sam.close()
