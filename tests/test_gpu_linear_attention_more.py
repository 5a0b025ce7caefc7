"""Linear attention: scales, values that are not finite, offsets past 31 bits, unusual lengths, and the example block.  Tolerances as in
test_gpu_linear_attention.py."""
import pytest
import torch

from tests.linear_attention_ref import norm2, recurrence, rel
from tests.test_gpu_linear_attention import STATE_TOL, TOL, TYPE, inputs, layer, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("scale", [-0.25, 0.0, 3.0])
@pytest.mark.parametrize("T", [5, 150])
def test_scales(handle, scale, T, dtype):
    q, k, v, ld, S = inputs(20, (2, T), 2, 2, 64, 64, dtype, 2)
    op = layer(handle, 2, T, 2, 64, 64, dtype=dtype, scale=scale)
    new = torch.empty_like(S)
    out = op.forward(q, k, v, ld, state=S, state_out=new)
    handle.synchronize()
    want, wantS = reference(q, k, v, ld, S, scale, [(0,), (1,)], range(2))
    assert rel(out, want) <= TOL[dtype] and rel(new, wantS) <= STATE_TOL
    op.close()


@pytest.mark.parametrize("dims", [(64, 64), (128, 128), (40, 24)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("where", ["v", "k", "q", "state"])
def test_values_that_are_not_finite(handle, where, dtype, dims):
    """They reach what the recurrence lets them reach, and nothing else: the tokens from theirs on up to the next reset (a query: its
    token alone), of their sequence and head."""
    dk, dv = dims
    T, bad, reset = 500, 130, 190
    q, k, v, ld, S = inputs(21, (2, T), 2, 2, dk, dv, dtype, 2)
    ld[0, reset, 1] = -float("inf")
    want, wantS = reference(q, k, v, ld, S, 1.0, [(0,), (1,)], range(2))
    if where == "state":
        S[0, 1, 3, 5] = float("inf")
        bad = 0
    else:
        {"q": q, "k": k, "v": v}[where][0, bad, 1, 3] = float("nan")
    op = layer(handle, 2, T, 2, dk, dv, dtype=dtype)
    new = torch.empty_like(S)
    out = op.forward(q, k, v, ld, state=S, state_out=new)
    handle.synchronize()
    assert rel(out[1], want[1]) <= TOL[dtype] and rel(out[0, :, 0], want[0, :, 0]) <= TOL[dtype]
    assert rel(out[0, reset:, 1], want[0, reset:, 1]) <= TOL[dtype]
    assert bad == 0 or rel(out[0, :bad, 1], want[0, :bad, 1]) <= TOL[dtype]
    assert not torch.isfinite(out[0, bad, 1]).all()
    if where == "q":
        assert torch.isfinite(out[0, bad + 1:, 1]).all()
    else:
        assert not torch.isfinite(out[0, bad:reset, 1]).all(-1).any()
    assert rel(new, wantS) <= STATE_TOL
    op.close()


@pytest.mark.parametrize("in_place", [False, True])
def test_not_finite_and_never_forgotten(handle, in_place):
    q, k, v, ld, S = inputs(22, (1, 400), 1, 1, 128, 128, "bf16", 1)
    v[0, 399, 0, 7] = float("inf")
    op = layer(handle, 1, 400, 1, 128, 128)
    new = S.clone() if in_place else torch.empty_like(S)
    out = op.forward(q, k, v, ld, state=new if in_place else S, state_out=new)
    handle.synchronize()
    clean = v.clone()
    clean[0, 399, 0, 7] = 0
    want, wantS = reference(q, k, clean, ld, S, 1.0, [(0,)], [0])
    assert rel(out[0, :399], want[0, :399]) <= TOL["bf16"]
    rest = torch.arange(128) != 7
    assert rel(out[0, 399, 0][rest.cuda()], want[0, 399, 0][rest]) <= TOL["bf16"]
    assert not torch.isfinite(out[0, 399, 0, 7]) and not torch.isfinite(new[0, 0, :, 7]).any()
    assert rel(new[0, 0][:, rest.cuda()], wantS[0, 0][:, rest]) <= STATE_TOL
    op.close()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_offsets_past_31_bits(handle, dtype):
    """A pool of more than 2^31 values, and sequences more than 2^31 values apart."""
    d, slots = 128, (1 << 31) // (128 * 128) + 3
    pool = torch.empty(slots, 1, d, d, device="cuda")
    q, k, v, ld, S = inputs(23, (2, 200), 1, 1, d, d, dtype, 2)
    at = [slots - 1, 1]
    pool[at] = S
    far = (1 << 31) + 64
    wide = torch.empty(far + 200 * d, device="cuda", dtype=TYPE[dtype])
    apart = wide.as_strided((2, 200, 1, d), (far, d, d, 1))
    apart.copy_(v)
    index = torch.tensor(at, dtype=torch.int32, device="cuda")
    op = layer(handle, 2, 200, 1, d, d, dtype=dtype)
    out = op.forward(q, k, apart, ld, state=pool, state_out=pool, slots=index)
    handle.synchronize()
    want, wantS = reference(q, k, v, ld, S, 1.0, [(0,), (1,)], range(2))
    assert rel(out, want) <= TOL[dtype] and rel(pool[at], wantS) <= STATE_TOL
    one = layer(handle, 2, 1, 1, d, d, dtype=dtype)
    got = one.step(q[:, 0], k[:, 0], v[:, 0], ld[:, 0], pool, slots=index)
    handle.synchronize()
    want, wantS = reference(q[:, :1], k[:, :1], v[:, :1], ld[:, :1], wantS, 1.0, [(0,), (1,)], range(2))
    assert rel(got, want[:, 0]) <= TOL[dtype] and rel(pool[at], wantS) <= 2 * STATE_TOL
    # and outputs that far apart
    del pool
    op.forward(q, k, v, ld, state=S, out=apart)
    handle.synchronize()
    want, _ = reference(q, k, v, ld, S, 1.0, [(0,), (1,)], range(2))
    assert rel(apart, want) <= TOL[dtype]
    op.close()
    one.close()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(40, 300, 8, 8, 64, 64), (3, 2000, 1, 1, 128, 64), (1, 5000, 3, 1, 64, 128), (200, 70, 2, 2, 32, 16), (1, 700, 2, 1, 200, 130)])
def test_many_short_and_few_long(handle, shape, dtype):
    """More sequences and heads than SMs, and so few that the axis of tokens is cut; ragged lengths of each."""
    B, T, H, Hk, dk, dv = shape
    lens = [T] + [(i * 7919) % (T + 1) for i in range(1, B)]
    q, k, v, ld, S = inputs(24, (B, T), H, Hk, dk, dv, dtype, B, decay=0.05)
    op = layer(handle, B, T, H, dk, dv, key_heads=Hk, dtype=dtype)
    new = torch.empty_like(S)
    out = op.forward(q, k, v, ld, state=S, state_out=new, lengths=torch.tensor(lens, dtype=torch.int32, device="cuda"))
    handle.synchronize()
    check = sorted({0, 1 % B, B // 2, B - 1})
    want, wantS = reference(q, k, v, ld, S, 1.0, [(b, slice(0, lens[b])) for b in check], check)
    for b in check:
        if lens[b]:
            assert rel(out[b, :lens[b]], want[b, :lens[b]]) <= TOL[dtype]
        assert rel(new[b], wantS[b]) <= STATE_TOL
    op.close()


@pytest.mark.parametrize("decay", [0.0, 1e-6, 1e-4])
def test_long_memories_do_not_drift(handle, decay):
    """Decays near 1 over thousands of tokens: rounding them would add up the same way at every token.  A hundred steps behind."""
    T, d = 6000, 64
    q, k, v, ld, S = inputs(25, (1, T + 100), 1, 1, d, d, "bf16", 1)
    ld = torch.full((1,), -decay, device="cuda")
    op = layer(handle, 1, T, 1, d, d)
    new = torch.empty_like(S)
    op.forward(q[:, :T], k[:, :T], v[:, :T], ld, state=S, state_out=new)
    for t in range(T, T + 100):
        op.step(q[:, t], k[:, t], v[:, t], ld, new)
    handle.synchronize()
    _, wantS = reference(q, k, v, ld.expand(1, T + 100, 1), S, 1.0, [(0,)], [0])
    assert rel(new, wantS) <= 1e-6          # sums of 6100 terms in fp32, in a tree and then 100 by ones: some 2^-24 each, at random
    op.close()


@pytest.mark.parametrize("dtype,limit", [("f32", 1e-4), ("bf16", 2e-2)])
def test_the_example_s_block(dtype, limit):
    """Steps against prompts through the whole block.  fp32: 3xTF32 connected layers of 512 terms (1e-5 each, two of them, through norms).
    bf16: queries, keys, values and the attention's output are rounded either way, its weights in the prompt only; a few 2^-8."""
    import importlib.util
    from pathlib import Path
    from nebula_b200 import api
    spec = importlib.util.spec_from_file_location("linear_attention_block", Path(__file__).resolve().parent.parent / "examples" / "linear_attention_block.py")
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    h = api.Handle(0, "tf32x3")
    out, state = example.run(h, batch=3, tokens=133, steps=3, width=256, heads=4, head_dim=64, dtype=dtype)
    assert out <= limit and state <= limit
    h.close()


def test_the_example_s_block_against_its_formulas():
    """A prompt through the block in fp32 against the same in 64 bits."""
    import importlib.util
    from pathlib import Path
    from nebula_b200 import api
    spec = importlib.util.spec_from_file_location("linear_attention_block", Path(__file__).resolve().parent.parent / "examples" / "linear_attention_block.py")
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    h = api.Handle(0, "fp32")
    b = example.Block(h, 128, 2, 64)
    x = torch.randn(2, 90, 128, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    state = b.state(2)
    s, y = b.forward(x, state, False)
    h.synchronize()
    d = {n: getattr(b, n).double().cpu() for n in ("w_in", "w_out", "norm_in", "norm_heads", "norm_out", "norm_next", "scale")}
    X = x.double().cpu().reshape(-1, 128)
    p = norm2(X, "rms", 1, d["norm_in"], None, 1e-6) @ d["w_in"].T
    q, k, v, gate = (p[:, i * 128:(i + 1) * 128].reshape(2, 90, 2, 64) for i in range(4))
    decay = torch.nn.functional.logsigmoid(p[:, 512:] + 3).reshape(2, 90, 2)
    outs, states = zip(*(recurrence(q[i], k[i] / 8, v[i], decay[i], torch.zeros(2, 64, 64, dtype=torch.float64), 1 / 8) for i in range(2)))
    o = norm2(torch.stack(outs).reshape(-1, 128), "rms", 2, d["norm_heads"], None, 1e-6)
    z = gate.reshape(-1, 128)
    o = (o * z * torch.sigmoid(z)) @ d["w_out"].T
    want = X + d["scale"] * norm2(o, "rms", 1, d["norm_out"], None, 1e-6)
    assert rel(s.view(-1, 128), want) <= 1e-5 and rel(y.view(-1, 128), norm2(want, "rms", 1, d["norm_next"], None, 1e-6)) <= 1e-5
    assert rel(state, torch.stack(states)) <= 1e-5
    b.close()
    h.close()
