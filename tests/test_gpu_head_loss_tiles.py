"""A head's loss and its gradients in every kind of tile of its logits: of 256, 192 and 128 hidden rows, with and without
tiles that are cut into stripes, over several stages of 64 columns, odd and even numbers of them and parts of one; and in
three pieces of the vocabulary and more. Bounds as in test_gpu_head_loss.py."""
import os
import subprocess

import pytest

from helpers import ROOT, twd
from test_gpu_head_loss import U, U16, check, make, reference

# vocab, d_model, rows, rows left out, softcap: width of a tile, tiles are cut, tiles are left whole
SHAPES = [
    ((1500, 1056, 350, 0, 30.0), (256, True, False)),
    ((12345, 1056, 1025, 0, 0.0), (256, False, True)),
    ((36001, 192, 1030, 0, 30.0), (256, False, True)),
    ((20003, 224, 1000, 231, 50.0), (256, True, True)),
    ((8200, 352, 1025, 0, 0.0), (192, False, True)),
    ((16500, 224, 1040, 15, 30.0), (192, False, True)),
    ((24001, 320, 700, 187, 30.0), (192, True, True)),
    ((4099, 160, 769, 0, 30.0), (128, False, True)),
    ((4099, 1056, 1000, 200, 0.0), (128, False, True)),
    ((50021, 96, 600, 0, 30.0), (128, False, True)),
    ((28001, 352, 513, 0, 0.0), (128, True, True)),
    ((33000, 288, 260, 60, 30.0), (128, True, True)),
]


def test_shapes_have_the_tiles_that_they_are_here_for(tmp_path):
    exe = tmp_path / "logit_tiles"
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wno-unknown-pragmas", "-I" + os.path.join(ROOT, "turbo-winfare-dense_amd", "csrc"),
                    os.path.join(ROOT, "tests", "cpp", "logit_tiles.cpp"), "-o", str(exe)], check=True, capture_output=True)
    sizes = [str(n) for (vocab, _, rows, out, _), _ in SHAPES for n in (rows - out, vocab)]
    lines = subprocess.run([str(exe)] + sizes, check=True, capture_output=True, text=True).stdout.split("\n")
    for ((vocab, d, rows, out, cap), kind), line in zip(SHAPES, lines):
        width, tiles, cut = (int(x) for x in line.split())
        assert (width, cut > 0, tiles > cut) == kind and d > 64 and rows > 128, (vocab, rows, line)
    # each width with whole tiles, cut ones, and odd and even numbers of stages
    for width in (256, 192, 128):
        assert {k[1:] for _, k in SHAPES if k[0] == width} >= {(False, True), (True, True)}
        assert {-(-s[1] // 64) % 2 for s, k in SHAPES if k[0] == width and k[2]} == {0, 1}


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [s for s, _ in SHAPES], ids=lambda s: "x".join(str(n) for n in s))
def test_loss_and_gradients(shape):
    import torch
    t = twd()
    vocab, d, rows, out, cap = shape
    h, w, targets, grad = make(vocab, d, rows, out, vocab + d)
    want, tol = reference(h, w, targets, cap, grad)
    loss = t.HeadLoss(rows, vocab, d, softcap=cap)
    losses, lse = loss.forward(h, w, targets)
    check("lse", lse, want["lse"], tol["lse"], U)
    check("losses", losses, want["losses"], tol["losses"], U)
    d_hidden, d_weight = loss.backward(h, w, targets, lse, grad=grad, d_weight=torch.empty(vocab, d, device="cuda:0"))
    check("d_hidden", d_hidden, want["d_hidden"], tol["d_hidden"], U16)
    check("d_weight", d_weight, want["d_weight"], tol["d_weight"], U)
    # the same bits again, and as bf16
    again = loss.backward(h, w, targets, lse, grad=grad)
    assert torch.equal(again[0], d_hidden) and torch.equal(again[1], d_weight.bfloat16())
    loss.close()


@pytest.mark.gpu
@pytest.mark.parametrize("vocab,d,rows,out,cap,pieces", [(5003, 96, 65536, 32768, 0.0, 3), (9999, 32, 65536, 40000, 30.0, 5),
                                                         (1000003, 96, 300, 20, 30.0, 3)])
def test_three_pieces_of_the_vocabulary_and_more(vocab, d, rows, out, cap, pieces):
    """A piece has at most 2^27 values of dz, in a multiple of 256 of the vocabulary."""
    import torch
    t = twd()
    most = (1 << 27) // rows // 256 * 256
    assert -(-(-(-vocab // 256) * 256) // most) == pieces
    h, w, targets, grad = make(vocab, d, rows, out, 12)
    want, tol = reference(h, w, targets, cap, grad)
    loss = t.HeadLoss(rows, vocab, d, softcap=cap)
    losses, lse = loss.forward(h, w, targets)
    check("lse", lse, want["lse"], tol["lse"], U)
    check("losses", losses, want["losses"], tol["losses"], U)
    base = torch.randn(vocab, d, device="cuda:0")
    d_weight = base.clone()
    d_hidden, _ = loss.backward(h, w, targets, lse, grad=grad, d_weight=d_weight, accumulate=True)
    check("d_hidden", d_hidden, want["d_hidden"], tol["d_hidden"], U16)
    check("d_weight", d_weight, base.double() + want["d_weight"], tol["d_weight"] + U * base.double().abs(), U)
    loss.close()
    del h, w, want, tol, d_hidden, d_weight, base
    torch.cuda.empty_cache()
