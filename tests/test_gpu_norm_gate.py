"""Norms before and after a block with its gate, residual scale and residual sum, against the formula in 64 bits.

Tolerances (2-norms).  fp32: sums of up to 32768 squares in fp32, in a tree, 1e-6 with what follows of a few roundings each
(2^-24 apiece), times the amplification of a cancelled mean (the inputs' mean is of the order of their deviation): 1e-5 as for the
framework's other fp32 results.  bf16: one rounding of the result, rms 2^-8/sqrt(3) at most."""
import pytest
import torch

from tests.linear_attention_ref import norm2, rel

pytestmark = pytest.mark.gpu
TOL = {"f32": 1e-5, "bf16": 2.0 ** -8 / 3 ** 0.5}
TYPE = {"f32": torch.float32, "bf16": torch.bfloat16}
GATES = {"linear": lambda z: z, "sigmoid": torch.sigmoid, "silu": lambda z: z * torch.sigmoid(z)}


def make(seed, rows, width, dtype, rdtype):
    g = torch.Generator().manual_seed(seed)
    x = (2 * torch.randn(rows, width, generator=g) + 0.5).to(TYPE[dtype])
    gate, res = (torch.randn(rows, width, generator=g) for _ in range(2))
    w = [1 + 0.2 * torch.randn(width, generator=g) for _ in range(5)]
    return x.cuda(), gate.to(TYPE[dtype]).cuda(), (3 * res).to(TYPE[rdtype]).cuda(), [t.cuda() for t in w]


def formula(x, norm, groups, eps, w, b, gate, act, cs, scale, res, nn, nw, nb):
    d = lambda t: None if t is None else t.double()  # noqa: E731
    u = norm2(d(x), norm, groups, d(w), d(b), eps)
    if gate is not None:
        u = u * GATES[act](d(gate))
    u = u * scale * (1 if cs is None else d(cs))
    if res is not None:
        u = u + d(res)
    return u, None if nn == "none" else norm2(u, nn, 1, d(nw), d(nb), eps)


CASES = [
    # rows, width, groups, norm, gate, residual, next
    (1, 1, 1, "rms", None, False, "none"), (1, 4096, 1, "rms", None, True, "rms"), (3, 128, 1, "layer", "silu", True, "layer"),
    (37, 2048, 16, "rms", "silu", False, "none"), (37, 2048, 16, "rms", "silu", True, "rms"), (5, 1000, 4, "layer", "sigmoid", True, "layer"),
    (9, 999, 3, "layer", "linear", True, "rms"), (130, 77, 7, "rms", None, False, "none"), (2, 8192, 1, "none", "silu", True, "rms"),
    (1, 32768, 1, "layer", "silu", True, "rms"), (2, 32767, 1, "rms", None, True, "layer"), (300, 40, 5, "layer", "silu", True, "layer"),
    (1000, 16, 2, "rms", "sigmoid", False, "none"), (2, 20000, 4, "rms", None, True, "rms"), (64, 1751, 1, "rms", "sigmoid", True, "none"),
    (3, 64, 64, "rms", None, False, "rms"), (400, 2056, 1, "rms", None, True, "rms"),
]


@pytest.mark.parametrize("types", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("case", CASES)
def test_norms(handle, case, types):
    rows, width, groups, norm, act, residual, nn = case
    dtype, rdtype = types
    x, gate, res, w = make(rows + width, rows, width, dtype, rdtype)
    gate, res = gate if act else None, res if residual else None
    bias = w[1] if norm == "layer" else None
    nb = w[4] if nn == "layer" else None
    s, y = handle.norm_gate_residual(x, w[0], bias, norm=norm, groups=groups, eps=1e-5, gate=gate, gate_act=act or "silu", residual=res, scale=0.5,
                                     channel_scale=w[2] if residual else None, next_norm=nn, next_weight=w[3] if nn != "none" else None, next_bias=nb)
    handle.synchronize()
    want, wanty = formula(x, norm, groups, 1e-5, w[0], bias, gate, act, w[2] if residual else None, 0.5, res, nn, w[3], nb)
    assert s.dtype == (TYPE[rdtype] if residual else x.dtype)
    assert rel(s, want) <= TOL[rdtype if residual else dtype]
    assert (y is None) == (nn == "none")
    if y is not None:
        assert rel(y, wanty) <= TOL[dtype]


@pytest.mark.parametrize("types", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("case", [
    (300, 866, 1, "rms", "silu", True, "none"), (300, 867, 1, "layer", "silu", True, "rms"), (301, 2046, 1, "rms", None, True, "layer"),
    (301, 2050, 1, "rms", "sigmoid", True, "rms"), (200, 2047, 1, "layer", None, False, "none"), (200, 2049, 1, "rms", "linear", True, "rms"),
    (300, 2, 1, "rms", None, True, "rms"), (300, 6, 3, "layer", "silu", True, "rms"), (200, 6, 2, "rms", None, True, "rms"),
    (150, 1000, 100, "rms", "silu", True, "layer"), (80, 32766, 1, "layer", "silu", True, "rms"),
])
def test_rows_in_pairs_and_single_values(handle, case, types):
    """Widths that are not whole 16-byte accesses, with enough rows that a thread has several."""
    test_norms(handle, case, types)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("width,skip", [(512, 0), (512, 8), (512, 3), (100, 1)])
def test_strided_rows_and_in_place(handle, width, skip, dtype):
    """Slices of wider tensors, aligned and not; the sum over the residual, y over x."""
    rows = 33
    wide, gate, res, w = make(2, rows, 2 * width + 16, dtype, dtype)
    x, gate, res = (t[:, skip:skip + width] for t in (wide, gate, res))
    w = [t[:width].contiguous() for t in w]
    want, wanty = formula(x, "rms", 1, 1e-6, w[0], None, gate, "silu", None, 1.0, res, "rms", w[3], None)
    around = wide.clone()
    s, y = handle.norm_gate_residual(x, w[0], gate=gate, residual=res, next_norm="rms", next_weight=w[3], out=res, y=x)
    handle.synchronize()
    assert s.data_ptr() == res.data_ptr() and y.data_ptr() == x.data_ptr()
    assert rel(s, want) <= TOL[dtype] and rel(y, wanty) <= TOL[dtype]
    around[:, skip:skip + width] = x
    assert torch.equal(around, wide)


def test_rows_of_zeros_and_of_huge_values(handle):
    x = torch.zeros(3, 256, device="cuda")
    x[1] = 1e18
    x[2, 5] = 1e-20
    s, y = handle.norm_gate_residual(x, norm="rms", next_norm="layer")
    handle.synchronize()
    want, wanty = formula(x, "rms", 1, 1e-6, None, None, None, None, None, 1.0, None, "layer", None, None)
    assert rel(s, want) <= TOL["f32"] and (s[0] == 0).all() and (y[0] == 0).all() and torch.isfinite(y).all()


def test_no_rows(handle):
    x = torch.zeros(0, 64, device="cuda")
    s, y = handle.norm_gate_residual(x, next_norm="rms")
    assert s.shape == y.shape == (0, 64)


def test_refusals(handle):
    from nebula_b200 import api
    x, gate, res, w = make(1, 4, 64, "bf16", "bf16")
    w = w[0]

    def refused(*a, code=1, **kw):
        with pytest.raises(api.NebulaError) as e:
            handle.norm_gate_residual(*a, **kw)
        assert e.value.code == code and len(str(e.value)) > 15

    refused(x.half(), w)
    refused(x, w[:32])
    refused(x, w.double())
    refused(x, w, gate=gate[:2])
    refused(x, w, gate=gate.float())
    refused(x, w, groups=5)
    refused(x, w, groups=0)
    refused(x, w, eps=-1.0)
    refused(x.t().contiguous().t(), w)
    refused(x, w, out=torch.empty(4, 64, device="cuda", dtype=torch.float16))
    refused(x.float(), w, residual=res, code=3)
    refused(torch.zeros(1, 32769, device="cuda"), code=3)
    lib = handle.lib
    assert lib.nb_norm_gate_residual(None, bytes(80), bytes(80)) == 1 and lib.nb_norm_gate_residual(handle.h, None, None) == 1
    s, _ = handle.norm_gate_residual(x, w)
    handle.synchronize()
    assert rel(s, formula(x, "rms", 1, 1e-6, w, None, None, None, None, 1.0, None, "none", None, None)[0]) <= TOL["bf16"]
