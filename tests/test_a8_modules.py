"""Modules with int8 codes and tokens in 8 bits (``a8``) when they are moved, copied, saved or loaded."""

from __future__ import annotations

import copy

import pytest
import torch

from llms_amd import kernels as fk
from llms_amd.kernels.quant import padded_rows
from tests.test_w8a8 import make

DEV = "cuda"
gpu = pytest.mark.gpu


def held(f):
    """Every int8 buffer of a module's a8 parts."""
    return [getattr(m, n) for m in f.modules() if getattr(m, "a8", False) for n in m.codes]


def odd_modules(device="cpu"):
    """An a8 Linear, FFN and attention with rows of 201 and 70 inputs, as from_eager builds them."""
    lin = fk.FusedLinear(201, 77)
    lin.int8 = lin.a8 = True
    lin.weight = None
    g = torch.Generator().manual_seed(0)
    lin.register_buffer("q", padded_rows(torch.randint(-127, 128, (77, 201), generator=g).to(torch.int8)))
    lin.register_buffer("s", torch.rand(77, generator=g))
    ffn = fk.TritonFFN.__new__(fk.TritonFFN)
    torch.nn.Module.__init__(ffn)
    ffn.int8 = ffn.a8 = True
    for n in ("qg", "qu"):
        ffn.register_buffer(n, padded_rows(torch.randint(-127, 128, (30, 70), generator=g).to(torch.int8)))
    ffn.down = lin
    return ffn.to(device)


def test_padded_rows_survive_a_move(tmp_path):
    """Codes at a stride of whole 16 bytes stay so when a module is moved, copied, saved or given a state."""
    f = odd_modules()
    want = [q.clone() for q in held(f)]
    assert len(want) == 3 and [q.stride(0) for q in held(f)] == [80, 80, 208]

    def check_held(m):
        assert [q.stride() for q in held(m)] == [(80, 1), (80, 1), (208, 1)] and all(map(torch.equal, held(m), want))

    check_held(f._apply(lambda t: t.clone(memory_format=torch.contiguous_format)))  # what .to(device) does
    check_held(copy.deepcopy(f))
    state = {k: v.contiguous() for k, v in f.state_dict().items()}
    for assign in (False, True):
        m = odd_modules()
        with torch.no_grad():
            for q in held(m):
                q.zero_()
        m.load_state_dict(state, assign=assign)
        check_held(m)
    torch.save(f, tmp_path / "m.pt")
    check_held(torch.load(tmp_path / "m.pt", weights_only=False))
    assert [q.stride(0) for q in held(odd_modules("meta"))] == [80, 80, 208]
    plain = fk.FusedLinear(201, 77)
    assert plain.to(torch.bfloat16).weight.dtype == torch.bfloat16


@gpu
@pytest.mark.parametrize("rows", [1, 40])
def test_moved_modules_answer_the_same(rows):
    lin = torch.nn.Linear(201, 77, bias=False, device=DEV, dtype=torch.bfloat16)
    f = fk.FusedLinear.from_linear(lin, int8=True, a8=True)
    x = make(rows, rows, 201, 1)[0].to(DEV)
    with torch.inference_mode():
        y = f(x)
        f = f.to("cpu").to(DEV)
        assert f.q.stride(0) == 208 and torch.equal(f(x), y)
