"""Linear attention with a decay for each head: prompts and single tokens against the recurrence in 64 bits.

Tolerances (2-norms).  State and fp32 outputs: fp32 arithmetic throughout, 1e-5 as for the framework's other fp32 results.  bf16
outputs: besides the one rounding of the output (relative error uniform within 2^-8, rms 2^-8/sqrt(3) at most) a term may pass one
bf16 rounding more on its way (the weight of a pair of tokens, or the state it is read through): two independent errors, rms
2^-8 * sqrt(2/3); the limit is 2^-8."""
import pytest
import torch

from tests.linear_attention_ref import recurrence, rel

pytestmark = pytest.mark.gpu
TOL = {"f32": 1e-5, "bf16": 2.0 ** -8}
STATE_TOL = 1e-5
TYPE = {"f32": torch.float32, "bf16": torch.bfloat16}


def inputs(seed, lead, H, Hk, dk, dv, dtype, slots, decay=0.3):
    g = torch.Generator().manual_seed(seed)
    t = TYPE[dtype]
    q = torch.randn(*lead, Hk, dk, generator=g).to(t)
    k = (torch.randn(*lead, Hk, dk, generator=g) / dk ** 0.5).to(t)
    v = torch.randn(*lead, H, dv, generator=g).to(t)
    ld = -decay * torch.rand(*lead, H, generator=g)
    S = torch.randn(slots, H, dk, dv, generator=g)
    return [x.cuda() for x in (q, k, v, ld, S)]


def reference(q, k, v, ld, S, scale, spans, slots):
    """spans: (index of a sequence's tokens in the leading dimensions) per sequence."""
    out = torch.zeros(v.shape, dtype=torch.float64)
    S = S.double().cpu().clone()
    c = [x.double().cpu() for x in (q, k, v, ld)]
    for at, slot in zip(spans, slots):
        out[at], S[slot] = recurrence(c[0][at], c[1][at], c[2][at], c[3][at], S[slot], scale)
    return out, S


def layer(handle, B, T, H, dk, dv, **kw):
    from nebula_b200 import api
    return api.LinearAttention(handle, B, T, H, dk, dv, **kw)


SHAPES = [
    # B, T, H, Hk, dk, dv
    (1, 1, 1, 1, 1, 1), (2, 1, 3, 3, 64, 64), (1, 2, 2, 1, 16, 32), (2, 17, 3, 3, 40, 72), (1, 63, 2, 2, 64, 64), (1, 64, 2, 2, 64, 64),
    (1, 65, 2, 2, 64, 64), (2, 128, 2, 2, 128, 128), (1, 129, 4, 2, 128, 128), (1, 200, 6, 2, 64, 128), (2, 191, 2, 1, 128, 64),
    (1, 300, 1, 1, 33, 57), (1, 130, 2, 2, 100, 20), (3, 97, 5, 5, 8, 8), (1, 150, 2, 2, 256, 256), (1, 77, 2, 2, 7, 250), (1, 500, 1, 1, 96, 80),
    (1, 1000, 2, 2, 128, 128), (1, 1537, 1, 1, 64, 64),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_prompts(handle, shape, dtype):
    B, T, H, Hk, dk, dv = shape
    q, k, v, ld, S = inputs(sum(shape), (B, T), H, Hk, dk, dv, dtype, B)
    op = layer(handle, B, T, H, dk, dv, key_heads=Hk, dtype=dtype, scale=dk ** -0.5)
    new = torch.full_like(S, float("nan"))
    out = op.forward(q, k, v, ld, state=S, state_out=new)
    handle.synchronize()
    want, wantS = reference(q, k, v, ld, S, dk ** -0.5, [(b,) for b in range(B)], range(B))
    assert rel(out, want) <= TOL[dtype]
    assert rel(new, wantS) <= STATE_TOL
    op.close()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("T", [1, 70, 700])
def test_no_state_and_no_decay(handle, T, dtype):
    """Starts from zeros, keeps no state, decays of 1: the plain sum over the prompt."""
    q, k, v, ld, S = inputs(T, (2, T), 2, 2, 64, 64, dtype, 2)
    op = layer(handle, 2, T, 2, 64, 64, dtype=dtype)
    out = op.forward(q, k, v)
    want, _ = reference(q, k, v, 0 * ld, 0 * S, 1.0, [(0,), (1,)], range(2))
    handle.synchronize()
    assert rel(out, want) <= TOL[dtype]
    new = torch.empty_like(S)
    op.forward(q, k, v, ld, state_out=new)
    _, wantS = reference(q, k, v, ld, 0 * S, 1.0, [(0,), (1,)], range(2))
    assert rel(new, wantS) <= STATE_TOL
    op.close()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("value", [-float("inf"), -200.0, -20.0])
def test_strong_decays(handle, value, dtype):
    """Tokens that forget everything before them, some next to one another, the first and the last of a chunk among them, with
    slow decays in between whose sums must keep their precision."""
    T = 300
    q, k, v, ld, S = inputs(5, (1, T), 2, 2, 64, 64, dtype, 1, decay=0.01)
    for t in (0, 1, 50, 63, 64, 100, 101, 127, 128, 191, 250, T - 1):
        ld[0, t, 0] = value
    ld[0, 140:200, 1] = value
    op = layer(handle, 1, T, 2, 64, 64, dtype=dtype)
    new = torch.empty_like(S)
    out = op.forward(q, k, v, ld, state=S, state_out=new)
    want, wantS = reference(q, k, v, ld, S, 1.0, [(0,)], [0])
    handle.synchronize()
    for h in range(2):
        assert rel(out[:, :, h], want[:, :, h]) <= TOL[dtype]
        assert rel(new[:, h], wantS[:, h]) <= STATE_TOL
    op.close()


def test_a_reset_forgets_infinities(handle):
    """What lies before a decay of zero does not reach what follows, not as inf * 0 either; later tokens never reach earlier ones."""
    T = 200
    q, k, v, ld, S = inputs(6, (1, T), 1, 1, 64, 64, "bf16", 1)
    ld[0, 70] = -float("inf")
    clean = v.clone()
    v[0, 30] = float("inf")
    v[0, 150] = float("nan")
    op = layer(handle, 1, T, 1, 64, 64)
    out = op.forward(q, k, v, ld, state=S)
    want, _ = reference(q, k, clean, ld, S, 1.0, [(0,)], [0])
    handle.synchronize()
    assert rel(out[0, :30], want[0, :30]) <= TOL["bf16"]
    assert rel(out[0, 70:150], want[0, 70:150]) <= TOL["bf16"]
    assert not torch.isfinite(out[0, 30:70]).any() and torch.isnan(out[0, 150:]).all()
    op.close()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dims", [(64, 64), (128, 128), (40, 72), (21, 33)])
def test_packed_sequences(handle, dims, dtype):
    """Lengths of zero, one, a chunk and around it, many chunks; slots out of order, one sequence not served."""
    dk, dv = dims
    lens = [0, 1, 64, 700, 0, 63, 65, 128, 129, 5]
    B, H, Hk = len(lens), 4, 2
    off = [sum(lens[:i]) for i in range(B + 1)]
    tokens = off[-1] + 9                    # rows behind the last sequence
    q, k, v, ld, S = inputs(7, (tokens,), H, Hk, dk, dv, dtype, 13)
    ld[off[3] + 100, 1] = -float("inf")
    slots = [12, 0, 3, 5, 7, 1, 2, -1, 9, 4]
    op = layer(handle, B, 700, H, dk, dv, key_heads=Hk, dtype=dtype, scale=0.5)
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    out = torch.full_like(v, 7.0)
    new = S.clone()
    op.forward(q, k, v, ld, state=new, state_out=new, offsets=dev(off), slots=dev(slots), out=out)
    handle.synchronize()
    served = [b for b in range(B) if slots[b] >= 0]
    want, wantS = reference(q, k, v, ld, S, 0.5, [(slice(off[b], off[b + 1]),) for b in served], [slots[b] for b in served])
    assert (out[off[-1]:] == 7).all() and (out[off[7]:off[8]] == 0).all()
    for b in served:
        if lens[b]:
            assert rel(out[off[b]:off[b + 1]], want[off[b]:off[b + 1]]) <= TOL[dtype]
        assert rel(new[slots[b]], wantS[slots[b]]) <= STATE_TOL
    for s in set(range(13)) - set(slots):
        assert torch.equal(new[s], S[s])
    assert torch.equal(new[12], S[12]) and torch.equal(new[7], S[7])        # sequences without tokens
    op.close()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_padded_sequences_of_any_layout(handle, dtype):
    """Time-major tensors, a head's tokens next to one another, slices of a wider projection, a decay a head; padding is not
    written, and what it holds is not read."""
    B, T, H, d = 3, 150, 2, 64
    lens = [150, 0, 77]
    q, k, v, ld, S = inputs(8, (B, T), H, H, d, d, dtype, B)
    for b in range(B):
        for x in (q, k, v):
            x[b, lens[b]:] = float("nan")
    ld = ld[0, 0].contiguous()
    want, wantS = reference(q, k, v, ld.expand(B, T, H), S, 1.0, [(b, slice(0, lens[b])) for b in range(B)], range(B))
    lengths = torch.tensor(lens, dtype=torch.int32, device="cuda")
    op = layer(handle, B, T, H, d, d, dtype=dtype)
    wide = torch.empty(B, T, H, 3 * d + 8, device="cuda", dtype=TYPE[dtype])
    wide[..., :d], wide[..., d:2 * d], wide[..., 2 * d:3 * d] = q, k, v
    odd = torch.empty(B, T, H, d + 1, device="cuda", dtype=TYPE[dtype])
    odd[..., 1:] = q
    layouts = [
        (q, k, v, torch.empty_like(v)),
        tuple(x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)) + (torch.empty(T, B, H, d, device="cuda", dtype=v.dtype).transpose(0, 1),),
        tuple(x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v)) + (torch.empty(B, H, T, d, device="cuda", dtype=v.dtype).transpose(1, 2),),
        (wide[..., :d], wide[..., d:2 * d], wide[..., 2 * d:3 * d], torch.empty_like(v)),
        (odd[..., 1:], k, v, torch.empty(B, T, H, d + 3, device="cuda", dtype=v.dtype)[..., 3:]),
    ]
    for lq, lk, lv, out in layouts:
        out.fill_(7.0)
        new = torch.empty_like(S)
        op.forward(lq, lk, lv, ld, state=S, state_out=new, lengths=lengths, out=out)
        handle.synchronize()
        for b in range(B):
            assert (out[b, lens[b]:] == 7).all()
            assert rel(out[b, :lens[b]], want[b, :lens[b]]) <= TOL[dtype]
        assert rel(new, wantS) <= STATE_TOL
    op.close()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 1), (1, 8, 8, 64, 64), (5, 3, 1, 128, 128), (3, 4, 2, 40, 72), (2, 2, 2, 33, 57), (300, 2, 2, 64, 96),
                                   (2, 2, 1, 256, 256), (7, 2, 2, 16, 130), (150, 4, 4, 9, 12)])
def test_steps(handle, shape, dtype):
    """Three tokens one by one, in place, then out of place."""
    B, H, Hk, dk, dv = shape
    q, k, v, ld, S = inputs(sum(shape), (B, 3), H, Hk, dk, dv, dtype, B)
    ld[B // 2, 1, H // 2] = -float("inf")
    op = layer(handle, B, 1, H, dk, dv, key_heads=Hk, dtype=dtype, scale=0.7)
    want, wantS = reference(q, k, v, ld, S, 0.7, [(b,) for b in range(B)], range(B))
    pool = S.clone()
    outs = [op.step(q[:, t], k[:, t], v[:, t], ld[:, t].contiguous(), pool) for t in range(2)]
    last = torch.empty_like(pool)
    before = pool.clone()
    outs.append(op.step(q[:, 2], k[:, 2], v[:, 2], ld[:, 2], pool, state_out=last))
    handle.synchronize()
    assert torch.equal(pool, before)
    assert rel(torch.stack(outs, 1), want) <= TOL[dtype]
    assert rel(last, wantS) <= STATE_TOL
    op.close()


def test_steps_on_slots(handle):
    B, H, d = 6, 2, 64
    q, k, v, ld, S = inputs(9, (B, 1), H, H, d, d, "bf16", 9)
    slots = [8, 0, -1, 3, 9, 5]
    op = layer(handle, B, 1, H, d, d)
    pool = S.clone()
    out = op.step(q[:, 0], k[:, 0], v[:, 0], ld[:, 0], pool, slots=torch.tensor(slots, dtype=torch.int32, device="cuda"))
    handle.synchronize()
    served = [0, 1, 3, 5]
    want, wantS = reference(q, k, v, ld, S, 1.0, [(b,) for b in served], [slots[b] for b in served])
    assert (out[[2, 4]] == 0).all() and rel(out[served], want[served, 0]) <= TOL["bf16"]
    for s in range(9):
        assert rel(pool[s], wantS[s]) <= STATE_TOL if s in slots else torch.equal(pool[s], S[s])
    op.close()


def test_a_prompt_and_its_continuation(handle):
    """A prompt in one piece, in two, and with its last tokens as steps give the same states and outputs."""
    T, H, d = 400, 2, 128
    q, k, v, ld, S = inputs(10, (1, T), H, H, d, d, "bf16", 1)
    whole, state = layer(handle, 1, T, H, d, d), torch.empty_like(S)
    out = whole.forward(q, k, v, ld, state_out=state)
    pool = torch.zeros_like(S)
    parts = []
    for a, b in ((0, 150), (150, 397)):
        op = layer(handle, 1, b - a, H, d, d)
        parts.append(op.forward(q[:, a:b], k[:, a:b], v[:, a:b], ld[:, a:b], state=pool, state_out=pool))
    for t in range(397, T):
        parts.append(whole.step(q[:, t], k[:, t], v[:, t], ld[:, t], pool)[:, None])
    handle.synchronize()
    assert rel(torch.cat(parts, 1), out) <= 2 * TOL["bf16"]
    assert rel(pool, state) <= 2 * STATE_TOL


def test_results_do_not_change_from_call_to_call(handle):
    q, k, v, ld, S = inputs(11, (1, 3000), 3, 3, 128, 128, "bf16", 1)
    op = layer(handle, 1, 3000, 3, 128, 128)
    op.prepare()
    got = []
    for _ in range(3):
        new = torch.empty_like(S)
        got.append((op.forward(q, k, v, ld, state=S, state_out=new), new))
    handle.synchronize()
    for out, new in got[1:]:
        assert torch.equal(out, got[0][0]) and torch.equal(new, got[0][1])
    want, wantS = reference(q, k, v, ld, S, 1.0, [(0,)], [0])
    assert rel(got[0][0], want) <= TOL["bf16"] and rel(got[0][1], wantS) <= STATE_TOL
    op.close()


def test_on_a_stream_of_its_own(handle):
    from nebula_b200 import api
    h = api.Handle(0)
    q, k, v, ld, S = inputs(12, (2, 500), 2, 2, 64, 64, "bf16", 2)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    h.set_stream(stream.cuda_stream)
    op = layer(h, 2, 500, 2, 64, 64)
    op.prepare()
    with torch.cuda.stream(stream):
        new = torch.empty_like(S)
        out = op.forward(q, k, v, ld, state=S, state_out=new)
        graph = torch.cuda.CUDAGraph()
        out2, new2 = torch.empty_like(out), torch.empty_like(S)
        with torch.cuda.graph(graph, stream=stream):
            op.forward(q, k, v, ld, state=S, state_out=new2, out=out2)
        graph.replay()
    h.synchronize()
    assert torch.equal(out, out2) and torch.equal(new, new2)
    want, _ = reference(q, k, v, ld, S, 1.0, [(0,), (1,)], range(2))
    assert rel(out, want) <= TOL["bf16"]
    del graph
    op.close()
    h.close()


def test_refusals(handle):
    from nebula_b200 import api
    B, T, H, d = 2, 10, 2, 64
    q, k, v, ld, S = inputs(13, (B, T), H, H, d, d, "bf16", B)
    op = layer(handle, B, T, H, d, d)
    ints = torch.zeros(B + 1, dtype=torch.int32, device="cuda")

    def refused(f, *a, code=1, **kw):
        with pytest.raises(api.NebulaError) as e:
            f(*a, **kw)
        assert e.value.code == code and len(str(e.value)) > 20

    for args in ((0, T, H, d, d), (B, 0, H, d, d), (B, T, 0, d, d), (B, T, H, 0, d), (B, T, H, d, -1)):
        refused(layer, handle, *args)
    refused(layer, handle, B, T, 3, d, d, key_heads=2)
    refused(layer, handle, B, T, H, 257, d, code=3)
    refused(layer, handle, B, T, H, d, 300, code=3)
    refused(op.forward, q.float(), k, v, ld)
    refused(op.forward, q[:, :5], k, v, ld)
    refused(op.forward, q, k, v, ld.double())
    refused(op.forward, q, k.cpu(), v, ld)
    refused(op.forward, q.transpose(2, 3).contiguous().transpose(2, 3), k, v, ld)
    refused(op.forward, q, k, v, ld, out=v)
    refused(op.forward, q, k, v, ld, state=S[:1])
    refused(op.forward, q, k, v, ld, state=S.bfloat16())
    refused(op.forward, q, k, v, ld, slots=ints[:B])
    refused(op.forward, q, k, v, ld, lengths=ints)
    refused(op.forward, q, k, v, ld, offsets=ints, lengths=ints[:B])
    refused(op.forward, q[0], k[0], v[0], ld[0], offsets=ints, lengths=ints[:B])
    refused(op.forward, q, k, v, ld, out=torch.empty(B, 1, H, d, device="cuda", dtype=v.dtype).expand(B, T, H, d))
    refused(op.step, q[:, 0], k[:, 0], v[:, 0], ld[:, 0], None)
    refused(op.step, q, k, v, ld, S)
    # the C entries without the Python checks
    lib = handle.lib
    assert lib.nb_linear_attention_forward(None, op._io) == 1 and lib.nb_linear_attention_forward(op.p, None) == 1
    assert lib.nb_linear_attention_step(op.p, None) == 1 and lib.nb_linear_attention_plan_create(handle.h, None, api.C.byref(api._VP())) == 1
    assert lib.nb_linear_attention_forward(op.p, bytes(216)) == 1
    fc = api.Connected(handle, 1, 8, 8)
    assert lib.nb_linear_attention_forward(fc.p, op._io) == 1
    assert lib.nb_fc_forward(op.p, None, None) == 1
    # and it still works
    out = op.forward(q, k, v, ld)
    want, _ = reference(q, k, v, ld, 0 * S, 1.0, [(0,), (1,)], range(B))
    handle.synchronize()
    assert rel(out, want) <= TOL["bf16"]
    fc.close()
    op.close()
