"""The ragged steps (several new tokens per sequence in packed rows) against
plain implementations in 64 bits: paged_attention_prep, paged_attention,
deltanet_decode_span and draft_verify, one by one and as one speculative step.

Tolerances count roundings: an output rounded to a type with machine epsilon e
is off by at most e/2 of its value; sums of n products in fp32 by n * 2^-24 of
the sum of their magnitudes; what each check adds to that is written beside it."""
import math

import numpy as np
import pytest
import torch

import spock_b200

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
F16, BF16 = torch.float16, torch.bfloat16


def _i32(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device=DEV)


def _starts(lens):
    return np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _half_step(t):
    return torch.finfo(t).eps / 2


class Cache:
    """A paged cache with randomly placed pages; slots behind the lengths and unused pages hold NaN."""

    def __init__(self, kv_lens, page, heads, dim, dtype, g, head_major=False, room=0):
        need = [-(-(n + room) // page) for n in kv_lens]
        n = sum(need) + 2
        shape = (n, heads, page, dim) if head_major else (n, page, heads, dim)
        self.k = torch.full(shape, math.nan, dtype=dtype, device=DEV)
        self.v = torch.full(shape, math.nan, dtype=dtype, device=DEV)
        if head_major:
            self.k, self.v = self.k.transpose(1, 2), self.v.transpose(1, 2)
        order = torch.randperm(n, device=DEV, generator=g).tolist()
        width = max(1, max(need))
        table = np.full((len(kv_lens), width), -1, np.int32)  # never read behind the lengths
        at = 0
        for b, m in enumerate(need):
            table[b, :m] = order[at:at + m]
            at += m
        self.table, self.len, self.page, self.lens = _i32(table), _i32(kv_lens), page, list(kv_lens)
        for b, n in enumerate(kv_lens):
            ids, slot = self.slots(b, torch.arange(n, device=DEV))
            self.k[ids, slot] = torch.randn(n, heads, dim, device=DEV, generator=g).to(dtype)
            self.v[ids, slot] = torch.randn(n, heads, dim, device=DEV, generator=g).to(dtype)

    def slots(self, b, p):
        return self.table[b].long()[p // self.page], p % self.page

    def args(self):
        return self.k, self.v, self.table, self.len


def _ref_attention(q, starts, c, scale, gate):
    """out, and the bound's ingredients per element: sum p |v| and the scores' error bound."""
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    mag, err = torch.zeros_like(out), torch.zeros_like(out)
    group, d = q.shape[1] // c.k.shape[2], q.shape[2]
    for b, (lo, hi) in enumerate(zip(starts[:-1], starts[1:])):
        n, length = int(hi - lo), c.lens[b]
        if n == 0 or length == 0:
            continue
        ids, slot = c.slots(b, torch.arange(length, device=DEV))
        last = length - n + torch.arange(n, device=DEV)
        hidden = torch.arange(length, device=DEV)[None] > last[:, None]
        for h in range(q.shape[1]):
            k, v = c.k[ids, slot, h // group].double(), c.v[ids, slot, h // group].double()
            x = q[lo:hi, h].double()
            s = (x @ k.T * scale).masked_fill(hidden, -math.inf)
            p = torch.softmax(s, -1)
            p = torch.where((last < 0)[:, None], 0.0, p)
            out[lo:hi, h], mag[lo:hi, h] = p @ v, p @ v.abs()
            # |s| is off by (d + 4) roundings of the products' magnitudes
            err[lo:hi, h] = ((d + 4) * 2.0 ** -24 * scale * (x.abs() @ k.abs().T).amax(-1))[:, None]
    if gate is not None:
        out, mag = out * torch.sigmoid(gate.double()), mag * torch.sigmoid(gate.double())
    return out, mag, err


def _check_attention(got, ref, mag, err):
    # the output's rounding; each weight rounded to the operand type, and the same in the sum that divides them
    # (e/2 + e/2 of sum p|v|); a score error of err moves a weight and the sum by err each; 2^-15 for exp, the
    # running rescale and sigmoid in fp32
    e = _half_step(got.dtype)
    tol = e * ref.abs() + (2 * e + 2 * err + 2.0 ** -15) * mag + 1e-30 + (6e-8 if got.dtype == F16 else 0)
    off = (got.double() - ref).abs()
    assert bool((off <= tol).all()), (float((off / tol).max()), int((~(off <= tol)).sum()))


ATTEND = [
    # dtype, head_dim, q_heads, kv_heads, page, new tokens, lengths
    (F16, 256, 8, 2, 16, [1], [1]),
    (F16, 256, 8, 2, 16, [1], [577]),
    (BF16, 256, 8, 2, 64, [1, 1, 1, 1], [1, 64, 65, 1000]),
    (F16, 256, 8, 2, 16, [5, 0, 3, 5, 1], [5, 40, 129, 900, 128]),
    (BF16, 256, 8, 2, 24, [5, 2, 7], [3, 0, 300]),              # more new tokens than positions: empty rows
    (F16, 256, 8, 2, 64, [300], [300]),
    (BF16, 256, 8, 2, 8, [129], [1000]),
    (F16, 128, 16, 4, 32, [33, 65, 1], [33, 193, 2047]),
    (BF16, 128, 8, 8, 256, [17, 1], [257, 513]),
    (F16, 64, 12, 4, 16, [43, 86, 1], [43, 500, 77]),           # 3 heads a group: 42 tokens a tile
    (BF16, 64, 8, 1, 128, [16, 1, 200], [4000, 1, 215]),
    (F16, 64, 128, 1, 16, [3], [130]),                          # 128 heads over one
    (F16, 256, 2, 2, 16, [1] * 300, [1 + 7 * i % 260 for i in range(300)]),
    (BF16, 128, 4, 4, 16, [1, 200, 1, 1], [5000, 200, 31, 4097]),
    (F16, 256, 8, 2, 128, [700], [2500]),
]


@pytest.mark.parametrize("case", range(len(ATTEND)))
@pytest.mark.parametrize("gated", [False, True])
def test_paged_attention(cuda_ok, case, gated):
    dtype, d, hq, hk, page, new, lens = ATTEND[case]
    g = _gen(case)
    c = Cache(lens, page, hk, d, dtype, g, head_major=case % 2 == 1)
    starts, total = _starts(new), sum(new)
    # q and gate where a projection leaves them, two more rows behind the last sequence
    rows = torch.randn(total + 2, hq, 2, d, device=DEV, generator=g).to(dtype)
    q, gate = rows[:, :, 0], rows[:, :, 1] if gated else None
    out = torch.full((total + 2, hq, d), 7.0, dtype=dtype, device=DEV)
    scale = 1 / math.sqrt(d)
    got = spock_b200.paged_attention(q, _i32(starts), *c.args(), scale, gate=gate, out=out)
    spock_b200.Context.get(0).sync()
    assert got is out and bool((out[total:] == 7.0).all())
    ref, mag, err = _ref_attention(q, starts, c, scale, gate)
    _check_attention(got[:total], ref[:total], mag[:total], err[:total])


def test_paged_attention_large_scores(cuda_ok):
    """Scores of some hundreds: the running maximum has to carry them, whichever tile holds it."""
    g = _gen(3)
    c = Cache([700, 700], 16, 2, 128, F16, g)
    for b, p in ((0, 3), (1, 650)):
        ids, slot = c.slots(b, torch.tensor([p], device=DEV))
        c.k[ids, slot] *= 8
    starts = _starts([4, 1])
    q = (torch.randn(5, 4, 128, device=DEV, generator=g) * 8).half()
    got = spock_b200.paged_attention(q, _i32(starts), *c.args(), 0.5)
    spock_b200.Context.get(0).sync()
    _check_attention(got, *_ref_attention(q, starts, c, 0.5, None))


def test_paged_attention_on_a_side_stream_and_in_a_graph(cuda_ok):
    """Two captured calls replayed in turn, each with its own workspace, and new lengths between replays."""
    g = _gen(4)
    c = Cache([900, 130], 16, 2, 256, F16, g)
    starts = _starts([2, 3])
    q = torch.randn(5, 8, 256, device=DEV, generator=g).half()
    q2 = torch.randn(5, 8, 256, device=DEV, generator=g).half()
    s, side = _i32(starts), torch.cuda.Stream()
    spock_b200.paged_attention(q, s, *c.args(), 0.0625)
    torch.cuda.synchronize()
    side.wait_stream(torch.cuda.current_stream())
    onside = spock_b200.paged_attention(q, s, *c.args(), 0.0625, stream=side)
    side.synchronize()
    graphs, outs = [], []
    for x in (q, q2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(spock_b200.paged_attention(x, s, *c.args(), 0.0625))
        graphs.append(gr)
    for lens in ([900, 130], [514, 129]):
        c.lens = lens
        c.len.copy_(_i32(lens))
        graphs[1].replay()
        graphs[0].replay()
        torch.cuda.synchronize()
        for x, o in ((q, outs[0]), (q2, outs[1])):
            _check_attention(o, *_ref_attention(x, starts, c, 0.0625, None))
        if lens[0] == 900:
            assert torch.equal(onside, outs[0])


def test_paged_attention_is_the_same_every_time(cuda_ok):
    g = _gen(5)
    lens = [1 + 37 * i % 3000 for i in range(40)]
    c = Cache(lens, 16, 2, 256, F16, g)
    q = torch.randn(40, 8, 256, device=DEV, generator=g).half()
    first = spock_b200.paged_attention(q, _i32(_starts([1] * 40)), *c.args(), 0.0625)
    for _ in range(5):
        assert torch.equal(first, spock_b200.paged_attention(q, _i32(_starts([1] * 40)), *c.args(), 0.0625))


def _table(n, rotary, theta=1e7):
    ang = np.arange(n)[:, None] * theta ** (-np.arange(rotary // 2) * 2.0 / rotary)
    return torch.tensor(np.stack([np.cos(ang), np.sin(ang)], -1), dtype=torch.float32, device=DEV)


def _ref_prep(x, w, rope, pos):
    y = x.double()
    if w is not None:
        y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + 1e-6) * (1 + w.double())
    if rope is None:
        return y
    r = rope.shape[1]
    cs = rope.double()[pos][:, None]
    lo, hi = y[..., :r], y[..., r:2 * r]
    return torch.cat([lo * cs[..., 0] - hi * cs[..., 1], hi * cs[..., 0] + lo * cs[..., 1], y[..., 2 * r:]], -1)


@pytest.mark.parametrize("dtype,d,hq,hk,page,rotary,gated,normed,new,lens", [
    (F16, 256, 8, 2, 16, 64, True, True, [1], [1]),
    (BF16, 256, 8, 2, 64, 64, True, True, [5, 0, 130, 1], [5, 9, 700, 65]),
    (F16, 128, 6, 2, 24, 128, False, True, [7, 1], [50, 24]),
    (BF16, 64, 4, 4, 8, 16, False, True, [3, 9], [3, 100]),
    (F16, 64, 4, 1, 128, 64, True, False, [200], [300]),
    (F16, 128, 8, 8, 16, 0, False, True, [2, 2], [17, 16]),
    (F16, 256, 8, 2, 16, 32, True, True, [1] * 1100, [1 + i % 40 for i in range(1100)]),
    (BF16, 256, 8, 2, 16, 64, True, True, [4, 2], [2, 5]),  # two tokens before position 0: skipped
])
def test_paged_attention_prep(cuda_ok, dtype, d, hq, hk, page, rotary, gated, normed, new, lens):
    g = _gen(7)
    c = Cache(lens, page, hk, d, dtype, g)
    starts, total = _starts(new), sum(new)
    width = hq * (2 if gated else 1) + 2 * hk
    # rows wider than what is read, two of them behind the last sequence
    proj = torch.randn(total + 2, width * d + 16, device=DEV, generator=g).to(dtype)[:, :width * d]
    qn, kn = ((torch.randn(d, device=DEV, generator=g) * 0.1).to(dtype) for _ in range(2)) if normed else (None, None)
    rope = _table(max(lens), rotary) if rotary else None
    before = c.k.clone(), c.v.clone()
    q_out = torch.full((total + 2, hq, d), 7.0, dtype=dtype, device=DEV)
    spock_b200.paged_attention_prep(proj, _i32(starts), *c.args(), rope=rope, q_norm=qn, k_norm=kn, gated=gated,
                                    q_out=q_out)
    spock_b200.Context.get(0).sync()
    x = proj[:total].reshape(total, width, d)
    pos = torch.cat([c.lens[b] - n + torch.arange(n, device=DEV) for b, n in enumerate(new)])
    heads = width - 2 * hk
    real = pos >= 0
    want_q = _ref_prep(x[:, :heads:2] if gated else x[:, :heads], qn, rope, pos.clamp(min=0))
    want_k = _ref_prep(x[:, heads:heads + hk], kn, rope, pos.clamp(min=0))
    # one rounding of the value; 2^-20 for the norm and the rotation in fp32, of the pair's magnitude (below 8)
    near = lambda a, b: bool(((a.double() - b).abs() <= _half_step(dtype) * b.abs() + 2.0 ** -17).all())
    assert near(q_out[:total][real], want_q[real])
    assert bool((q_out[total:] == 7.0).all()) and bool((q_out[:total][~real] == 7.0).all())
    k_ref, v_ref, touched = before[0].double(), before[1].clone(), torch.zeros(c.k.shape[:2], dtype=torch.bool, device=DEV)
    for b, (lo, hi) in enumerate(zip(starts[:-1], starts[1:])):
        keep = torch.arange(lo, hi, device=DEV)[real[lo:hi]]
        ids, slot = c.slots(b, pos[keep])
        k_ref[ids, slot], v_ref[ids, slot] = want_k[keep], x[keep, heads + hk:]
        touched[ids, slot] = True
    assert near(c.k[touched], k_ref[touched])
    assert torch.equal(c.k[~touched].view(torch.int16), before[0][~touched].view(torch.int16))
    assert torch.equal(c.v.contiguous().view(torch.int16), v_ref.contiguous().view(torch.int16))


def _span_inputs(new, heads, seed, extra=0):
    g = _gen(seed)
    total, b = sum(new) + extra, len(new)
    half = lambda *s, sd=1.0: (torch.randn(*s, device=DEV, generator=g) * sd).half()
    row = half(total, heads * 512 + 2 * heads)
    qkv, z, a, bb = row.split([heads * 384, heads * 128, heads, heads], 1)
    layer = spock_b200.DeltaNetLayer(
        half(heads * 384, 4, sd=0.5),
        torch.stack([torch.rand(heads, device=DEV, generator=g) * 3 - 2,
                     torch.randn(heads, device=DEV, generator=g) * 0.1], 1).contiguous(),
        1 + 0.1 * torch.randn(128, device=DEV, generator=g), num_heads=heads)
    conv = half(b, heads * 384, 4)
    state = torch.randn(b, heads, 128, 128, device=DEV, generator=g) * 0.05
    return layer, qkv, conv, state, a, bb, z


def _ref_span(layer, qkv, conv, state, a, b, z, starts, counts):
    h = layer.num_heads
    a_log, dt = layer.a_log_bias.double().unbind(1)
    out = torch.zeros(qkv.shape[0], h * 128, dtype=torch.float64, device=DEV)
    states, convs = state.double().clone(), conv.double().clone()
    w = layer.conv_weight.double()
    for s in range(len(starts) - 1):
        for t in range(starts[s], starts[s] + counts[s]):
            convs[s] = torch.cat([convs[s][:, 1:], qkv[t].double()[:, None]], 1)
            y = (convs[s] * w).sum(1)
            q, k, v = (y * torch.sigmoid(y)).reshape(3, h, 128)
            q = q / torch.sqrt(q.square().sum(-1, keepdim=True) + 1e-6)
            k = k / torch.sqrt(k.square().sum(-1, keepdim=True) + 1e-6)
            step = -torch.exp(a_log) * torch.nn.functional.softplus(a[t].double() + dt, threshold=1e9)
            states[s] *= torch.exp(step)[:, None, None]
            delta = torch.sigmoid(b[t].double())[:, None] * (v - torch.einsum("hk,hkv->hv", k, states[s]))
            states[s] += torch.einsum("hk,hv->hkv", k, delta)
            o = torch.einsum("hk,hkv->hv", q, states[s]) / math.sqrt(128)
            o = o / torch.sqrt(o.square().mean(-1, keepdim=True) + layer.eps) * layer.norm_weight.double()
            g = z[t].double().reshape(h, 128)
            out[t] = (o * g * torch.sigmoid(g)).reshape(-1)
    return out, states, convs


def _check_span_out(got, ref):
    # fp16's rounding, and an absolute part: o before its norm is a sum of 128 products (128 roundings of 2^-24)
    # after up to 20 state updates, each likewise; the norm divides by an rms of the same sums, so 2^-24 * 128 * 20 *
    # (largest normed value, below 16 after w and the gate) bounds it. Subnormal fp16 steps are 2^-24.
    tol = _half_step(F16) * ref.abs() + 128 * 20 * 16 * 2.0 ** -24 * 0.25
    assert bool(((got.double() - ref).abs() <= tol).all()), float(((got.double() - ref).abs() / tol).max())


def _check_span_state(got, ref):
    # relative to the state's largest entry: 20 updates of (decay, 128-term product, add), 132 roundings each
    tol = 20 * 132 * 2.0 ** -24 * float(ref.abs().max())
    assert float((got.double() - ref).abs().max()) <= tol


@pytest.mark.parametrize("new,heads", [([1], 16), ([5, 5, 5], 16), ([3, 0, 8, 1, 9], 4), ([17, 20], 2),
                                       ([1 + i % 6 for i in range(40)], 16)])
def test_deltanet_decode_span(cuda_ok, new, heads):
    layer, qkv, conv, state, a, b, z = _span_inputs(new, heads, seed=len(new), extra=2)
    starts, total = _starts(new), sum(new)
    s = _i32(starts)
    ctx = spock_b200.Context.get(0)
    saved = state.clone(), conv.clone(), qkv.clone()
    # verification: outputs of all rows, nothing else changes
    out = torch.full((total + 2, heads * 128), 7.0, dtype=F16, device=DEV)
    spock_b200.deltanet_decode_span(layer, qkv, conv, state, a, b, z, s, out=out)
    ctx.sync()
    ref, ref_state, ref_conv = _ref_span(layer, qkv, conv, state, a, b, z, starts, new)
    _check_span_out(out[:total], ref[:total])
    assert bool((out[total:] == 7.0).all())
    assert torch.equal(state, saved[0]) and torch.equal(conv, saved[1]) and torch.equal(qkv, saved[2])
    # outputs and state at once
    st, cv = torch.full_like(state, math.nan), torch.full_like(conv, math.nan)
    out2 = torch.empty_like(out)
    spock_b200.deltanet_decode_span(layer, qkv, conv, state, a, b, z, s, out=out2, state_out=st, conv_out=cv)
    ctx.sync()
    assert torch.equal(out2[:total], out[:total])
    _check_span_state(st, ref_state)
    assert torch.equal(cv.double(), ref_conv)
    # commit of the first counts rows (more than there are: all; negative: none), in place
    counts = [(0, 1, n // 2, n, n + 3, -1)[i % 6] for i, n in enumerate(new)]
    take = [max(0, min(c, n)) for c, n in zip(counts, new)]
    _, ref_state, ref_conv = _ref_span(layer, qkv, conv, state, a, b, z, starts, take)
    spock_b200.deltanet_decode_span(layer, qkv, conv, state, a, b, None, s, counts=_i32(counts), state_out=state,
                                    conv_out=conv)
    ctx.sync()
    _check_span_state(state, ref_state)
    assert torch.equal(conv.double(), ref_conv)
    none = torch.tensor([t == 0 for t in take], device=DEV)
    assert torch.equal(state[none], saved[0][none])


def test_deltanet_decode_span_taken_rows_only(cuda_ok):
    layer, qkv, conv, state, a, b, z = _span_inputs([4, 6], 4, seed=1)
    out = torch.full((10, 512), 7.0, dtype=F16, device=DEV)
    spock_b200.deltanet_decode_span(layer, qkv, conv, state, a, b, z, _i32([0, 4, 10]), counts=_i32([2, 9]), out=out)
    ref, _, _ = _ref_span(layer, qkv, conv, state, a, b, z, [0, 4, 10], [2, 6])
    taken = torch.tensor([1, 1, 0, 0] + [1] * 6, device=DEV).bool()
    _check_span_out(out[taken], ref[taken])
    assert bool((out[~taken] == 7.0).all())


def test_deltanet_decode_span_extreme_gates(cuda_ok):
    """Decays of 0 and 1 and write strengths of 0 and 1: a = b = +-60000."""
    layer, qkv, conv, state, a, b, z = _span_inputs([6, 6], 4, seed=2)
    a[1::3], a[2::3] = 60000.0, -60000.0
    b[::2], b[1::4] = -60000.0, 60000.0
    st, cv = torch.empty_like(state), torch.empty_like(conv)
    out = torch.empty(12, 512, dtype=F16, device=DEV)
    spock_b200.deltanet_decode_span(layer, qkv, conv, state, a, b, z, _i32([0, 6, 12]), out=out, state_out=st,
                                    conv_out=cv)
    spock_b200.Context.get(0).sync()
    ref, ref_state, _ = _ref_span(layer, qkv, conv, state, a, b, z, [0, 6, 12], [6, 6])
    _check_span_state(st, ref_state)
    # where o is nothing but rounding (the state decayed to zero and nothing written) the norm divides noise
    fine = torch.isfinite(out) & (ref.abs() > 0)
    assert bool(torch.isfinite(out).all())
    _check_span_out(out[fine], ref[fine])


def test_deltanet_decode_span_matches_single_steps(cuda_ok):
    """A span equals the framework's single-token step applied token by token, within that step's extra roundings."""
    n, heads = 4, 16
    layer, qkv, conv, state, a, b, z = _span_inputs([n, n], heads, seed=9)
    starts = _i32([0, n, 2 * n])
    st, cv = torch.empty_like(state), torch.empty_like(conv)
    out = torch.empty(2 * n, 2048, dtype=F16, device=DEV)
    spock_b200.deltanet_decode_span(layer, qkv, conv, state, a, b, z, starts, out=out, state_out=st, conv_out=cv)
    state1, conv1 = state.clone(), conv.clone()
    for t in range(n):
        pick = lambda x: x[[t, n + t]].contiguous()
        o = spock_b200.deltanet_decode_step(layer, pick(qkv), conv1, state1, pick(a), pick(b), pick(z))
        # the step stores the conv output, q and k in fp16: 3 roundings of 2^-11 on each side of a product
        assert float((o.float() - out[[t, n + t]].float()).abs().max()) <= 8 * 2.0 ** -11 * float(o.abs().max())
    assert torch.equal(conv1, cv)
    assert float((state1 - st).abs().max()) <= 4 * n * 2.0 ** -11 * float(st.abs().max())


def _ref_verify(logits, tokens, starts, u_acc, u_smp, temp, probs):
    x = logits.double().cpu()
    x = torch.where(torch.isnan(x), -math.inf, x)
    tokens, emitted, out = tokens.tolist(), [], [-5] * logits.shape[0]
    for b, (lo, hi) in enumerate(zip(starts[:-1], starts[1:])):
        if lo == hi:
            emitted.append(0)
            continue
        t = 1.0 if temp is None else float(temp[b])
        i = lo
        while True:
            best = int(torch.nonzero(x[i] == x[i].max())[0])
            if t > 0:
                e = torch.where(x[i] == x[i].max(), 0.0, (x[i] - x[i].max()) / t).exp()
                e = torch.where(x[i] == -math.inf, 0.0, e)
                p = e / e.sum() if float(e.sum()) > 0 else e
                w = p
            if i == hi - 1:
                break
            d = tokens[i + 1]
            if t > 0:
                qd = 1.0 if probs is None else float(probs[i, d])
                if not float(u_acc[i]) * qd < float(p[d]):
                    w = p.clone()
                    if probs is None:
                        w[d] = 0
                    else:
                        w = (p - probs[i].double().cpu()).clamp(min=0)
                    w = w if float(w.sum()) > 0 else p
                    break
            elif best != d:
                break
            out[i] = d
            i += 1
        if t > 0:
            c = w.cumsum(0)
            over = torch.nonzero((c > float(u_smp[b]) * c[-1]) & (w > 0))
            best = int(over[0]) if len(over) else int(torch.nonzero(w > 0)[-1]) if bool((w > 0).any()) else 0
        out[i] = best
        out[i + 1:hi] = [-1] * (hi - i - 1)
        emitted.append(i - lo + 1)
    return emitted, out


def _verify_inputs(rows, vocab, dtype, seed, probs, spread=3.0):
    g = _gen(seed)
    total = sum(rows)
    logits = (torch.randn(total, vocab, device=DEV, generator=g) * spread).to(dtype)
    tokens = torch.randint(0, vocab, (total,), device=DEV, generator=g)
    q = None
    if probs:
        q = torch.softmax(logits.float() + 0.7 * torch.randn(total, vocab, device=DEV, generator=g), -1)
        drafted = torch.multinomial(q, 1, generator=g)[:, 0]
    else:
        drafted = torch.where(torch.rand(total, device=DEV, generator=g) < 0.7, logits.float().argmax(-1), tokens)
    tokens[1:] = drafted[:-1]
    return (logits, tokens.int(), torch.rand(total, device=DEV, generator=g),
            torch.rand(len(rows), device=DEV, generator=g), q)


def _run_verify(logits, tokens, starts, ua, us, temp, probs):
    out = torch.full((logits.shape[0],), -5, dtype=torch.int32, device=DEV)
    emitted, out = spock_b200.draft_verify(logits, tokens, _i32(starts), ua, us, temp, probs, out_tokens=out)
    spock_b200.Context.get(0).sync()
    return emitted.tolist(), out.tolist()


@pytest.mark.parametrize("dtype", [F16, BF16, torch.float32])
@pytest.mark.parametrize("vocab,rows", [(1, [3]), (5, [1, 4]), (1000, [5] * 20), (32003, [1, 9, 0, 4, 6]),
                                        (248320, [5, 3])])
@pytest.mark.parametrize("probs", [False, True])
def test_draft_verify(cuda_ok, dtype, vocab, rows, probs):
    logits, tokens, ua, us, q = _verify_inputs(rows, vocab, dtype, vocab + len(rows), probs)
    starts = _starts(rows)
    heat = torch.tensor([(1.0, 0.0, 0.7, 1.6)[i % 4] for i in range(len(rows))], device=DEV)
    for temp in (None, heat):
        assert _run_verify(logits, tokens, starts, ua, us, temp, q) == \
            _ref_verify(logits, tokens, starts, ua, us, temp, q)


def test_draft_verify_strided_rows_behind_the_last(cuda_ok):
    """Rows of an odd stride at an odd offset; two rows behind the last sequence stay as they are."""
    logits, tokens, ua, us, q = _verify_inputs([4, 3, 2], 1001, F16, 5, True)
    wide = torch.full((9, 1007), 60000.0, dtype=F16, device=DEV)
    wide[:, 3:1004] = logits
    wq = torch.full((9, 1003), 9.0, device=DEV)
    wq[:, 1:1002] = q
    starts = [0, 4, 7]
    got = _run_verify(wide[:, 3:1004], tokens, starts, ua, us[:2].contiguous(), None, wq[:, 1:1002])
    assert got == _ref_verify(logits, tokens, starts, ua, us, None, q)
    assert got[1][7:] == [-5, -5]


def test_draft_verify_borders(cuda_ok):
    """Numbers that fall on a border exactly: equal weights, powers of two, u = 0, the largest u below 1."""
    vocab = 4096
    logits = torch.zeros(3 * 7, vocab, dtype=F16, device=DEV)
    tokens = torch.full((21,), 9, dtype=torch.int32, device=DEV)
    ua = torch.full((21,), 1.0, device=DEV)
    ua[0::3] = 2.0 ** -12                       # p = 2^-12: u q < p fails on equality ...
    ua[3::6] = float(np.nextafter(np.float32(2.0 ** -12), np.float32(0)))  # ... and holds just below
    us = torch.tensor([0.0, 0.5, 0.25, float(np.nextafter(np.float32(1), np.float32(0))), 2.0 ** -12, 0.75, 9 / 4096],
                      device=DEV)
    starts = _starts([3] * 7)
    assert _run_verify(logits, tokens, starts, ua, us, None, None) == \
        _ref_verify(logits, tokens, starts, ua, us, None, None)
    q = torch.full((21, vocab), 2.0 ** -12, device=DEV)  # the draft's own distribution: the rest is zero everywhere
    ua = torch.full((21,), 1.0, device=DEV)
    assert _run_verify(logits, tokens, starts, ua, us, None, q) == \
        _ref_verify(logits, tokens, starts, ua, us, None, q)


def test_draft_verify_masked_logits(cuda_ok):
    """-inf, the type's lowest value, NaN and +inf among the logits; a row with nothing left; ties of the maximum."""
    logits, tokens, ua, us, q = _verify_inputs([2] * 8, 777, F16, 6, False)
    logits[0, 100:] = -math.inf
    logits[2, :776] = torch.finfo(F16).min
    logits[4, ::2] = math.nan
    logits[6, [30, 400]] = math.inf
    logits[8] = -math.inf
    logits[10, [5, 6, 700]] = 30.0
    logits[12] = math.nan
    starts = _starts([2] * 8)
    for temp in (None, torch.zeros(8, device=DEV)):
        got = _run_verify(logits, tokens, starts, ua, us, temp, None)
        if temp is not None:
            logits[[8, 12]] = torch.tensor([[0.0] * 777], device=DEV).half()  # nothing left: index 0 by definition
        assert got == _ref_verify(logits, tokens, starts, ua, us, temp, None)


def test_bad_device_data_is_reported_not_used(cuda_ok):
    """Page ids, lengths, starts and token ids out of range: the kernels skip them and the next sync says so."""
    ctx = spock_b200.Context.get(0)
    g = _gen(8)

    def refused():
        with pytest.raises(spock_b200.SpockError) as e:
            ctx.sync()
        assert e.value.code == spock_b200.SPOCK_ERR_INVALID
        ctx.sync()

    c = Cache([300, 40], 16, 2, 256, F16, g)
    q = torch.randn(4, 8, 256, device=DEV, generator=g).half()
    proj = torch.randn(4, 5120, device=DEV, generator=g).half()
    starts = _i32([0, 2, 4])
    good = c.table.clone(), c.len.clone()
    for bad in (-1, c.k.shape[0], 2 ** 31 - 1):
        c.table.copy_(good[0])
        ref = _ref_attention(q, [0, 2, 4], c, 0.0625, None)  # the prep below writes new rows each time
        c.table[0, 18] = bad
        out = spock_b200.paged_attention(q, starts, *c.args(), 0.0625)
        refused()
        _check_attention(out[2:], *(t[2:] for t in ref))  # the other sequence is none the worse
        spock_b200.paged_attention_prep(proj, starts, *c.args(), gated=True)
        refused()
    c.table.copy_(good[0])
    c.len[1] = 16 * c.table.shape[1] + 1  # more positions than the table has pages for
    spock_b200.paged_attention(q, starts, *c.args(), 0.0625)
    refused()
    spock_b200.paged_attention_prep(proj, starts, *c.args(), gated=True)
    refused()
    c.len.copy_(good[1])
    spock_b200.paged_attention_prep(proj, starts, *c.args(), gated=True, rope=_table(40, 64))
    refused()  # position 298 and a table of 40
    for s in ([0, 3, 2], [0, 2, 5], [-1, 2, 4]):
        spock_b200.paged_attention(q, _i32(s), *c.args(), 0.0625)
        refused()
    layer, qkv, conv, state, a, b, z = _span_inputs([2, 2], 4, seed=1)
    spock_b200.deltanet_decode_span(layer, qkv, conv, state, a, b, z, _i32([0, 2, 9]))
    refused()
    logits, tokens, ua, us, _ = _verify_inputs([2, 2], 100, F16, 1, False)
    tokens[1] = 100
    emitted, _ = spock_b200.draft_verify(logits, tokens, starts, ua, us)
    refused()
    assert emitted[0] == 1
    tokens[1] = 5
    spock_b200.draft_verify(logits, tokens, _i32([0, 2, 9]), ua, us)
    refused()


def test_paged_attention_refuses(cuda_ok):
    g = _gen(1)
    c = Cache([20], 16, 2, 64, F16, g)
    q = torch.zeros(1, 8, 64, dtype=F16, device=DEV)
    s = _i32([0, 1])

    def refused(code, text, **change):
        a = dict(q=q, start=s, k_pages=c.k, v_pages=c.v, page_table=c.table, kv_len=c.len, scale=1.0)
        a.update(change)
        with pytest.raises(spock_b200.SpockError, match=text) as e:
            spock_b200.paged_attention(**a)
        assert e.value.code == code

    bad, unsup = spock_b200.SPOCK_ERR_INVALID, spock_b200.SPOCK_ERR_UNSUPPORTED
    odd = torch.zeros(4, 12, 2, 64, dtype=F16, device=DEV)
    refused(unsup, "page_size must be a multiple of 8", k_pages=odd, v_pages=odd)
    wide = torch.zeros(4, 16, 2, 96, dtype=F16, device=DEV)
    refused(unsup, "head_dim is 64, 128 or 256", k_pages=wide, v_pages=wide,
            q=torch.zeros(1, 8, 96, dtype=F16, device=DEV))
    refused(bad, "q_heads must be a multiple", q=torch.zeros(1, 7, 64, dtype=F16, device=DEV))
    refused(unsup, "at most 128", q=torch.zeros(1, 258, 64, dtype=F16, device=DEV))
    refused(bad, "same shape and strides", v_pages=c.v[:3])
    refused(bad, "disagree on the batch", kv_len=_i32([20, 20]))
    refused(bad, "16-byte aligned", q=torch.zeros(513, dtype=F16, device=DEV)[1:].view(1, 8, 64))
    refused(bad, "workspace too small", workspace=torch.zeros(8, dtype=torch.uint8, device=DEV))
    refused(bad, "expected a tensor on", start=torch.tensor([0, 1], dtype=torch.int32))
    refused(bad, "expected the shape of q", gate=torch.zeros(1, 8, 128, dtype=F16, device=DEV))
    refused(bad, "multiples of 8", q=torch.zeros(1, 8, 65, dtype=F16, device=DEV)[..., :64])
    slim = torch.zeros(4, 16, 2, 72, dtype=F16, device=DEV)[..., :64]
    refused(bad, "head strides of 64", k_pages=slim, v_pages=slim)
    # no rows at all is a call like any other
    assert spock_b200.paged_attention(q[:0], _i32([0, 0]), *c.args(), 1.0).shape == (0, 8, 64)


def test_other_ragged_steps_refuse(cuda_ok):
    g = _gen(1)
    bad, unsup = spock_b200.SPOCK_ERR_INVALID, spock_b200.SPOCK_ERR_UNSUPPORTED

    def refused(code, text, f, *a, **k):
        with pytest.raises(spock_b200.SpockError, match=text) as e:
            f(*a, **k)
        assert e.value.code == code

    c, s = Cache([20], 16, 2, 64, F16, g), _i32([0, 1])
    proj = torch.zeros(1, 12 * 64, dtype=F16, device=DEV)
    prep = spock_b200.paged_attention_prep
    refused(bad, "q heads", prep, proj[:, :700], s, *c.args())
    refused(bad, "q heads", prep, proj[:, :7 * 64], s, *c.args(), gated=True)
    refused(bad, "bad arguments", prep, proj, s, *c.args(), q_norm=torch.zeros(64, dtype=F16, device=DEV))
    refused(unsup, "rotary must be a multiple", prep, proj, s, *c.args(), rope=_table(30, 2))
    refused(bad, "head_dim elements", prep, proj, s, *c.args(), q_norm=torch.zeros(32, dtype=F16, device=DEV),
            k_norm=torch.zeros(64, dtype=F16, device=DEV))
    layer, qkv, conv, state, a, b, z = _span_inputs([2], 4, seed=1)
    span, s = spock_b200.deltanet_decode_span, _i32([0, 2])
    refused(bad, "go together", span, layer, qkv, conv, state, a, b, z, s, state_out=state)
    refused(bad, "expected a tensor of shape", span, layer, qkv[:, :500], conv, state, a, b, z, s)
    refused(bad, "NULL pointer", span, layer, qkv, conv, state, a, b, None, s)
    refused(bad, "same row stride", span, layer, qkv, conv, state, a, b.contiguous(), z, s)
    x = torch.zeros(2, 10, dtype=F16, device=DEV)
    u = torch.zeros(2, device=DEV)
    refused(bad, "a value per row", spock_b200.draft_verify, x, _i32([1, 2]), s, u, u)
    refused(bad, "workspace too small", spock_b200.draft_verify, x, _i32([1, 2]), s, u, u[:1],
            workspace=torch.zeros(16, dtype=torch.uint8, device=DEV))


def test_one_speculative_step(cuda_ok):
    """The four steps as a server runs them: two rounds of drafts through one attention layer and one DeltaNet layer,
    the accepted tokens committed; after each, the caches equal those of the accepted tokens taken one by one."""
    g = _gen(11)
    heads, hidden, vocab, nseq = 4, 64, 50, 3
    layer, _, conv, state, *_ = _span_inputs([1] * nseq, heads, seed=11)
    w = lambda o, i: (torch.randn(o, i, device=DEV, generator=g) * 0.2).half()
    emb, w_attn, w_dn, head = w(vocab, hidden) * 4, w((2 * 4 + 2 * 2) * 64, hidden), w(heads * 514, hidden), \
        w(vocab, 4 * 64 + heads * 128)
    qn = kn = torch.zeros(64, dtype=F16, device=DEV)
    rope = _table(64, 32)
    page, width = 8, 8
    kp = torch.full((nseq * width, page, 2, 64), math.nan, dtype=F16, device=DEV)
    vp = kp.clone()
    table = torch.randperm(nseq * width, device=DEV, generator=g).int().reshape(nseq, width)
    length = _i32([0] * nseq)

    def forward(tokens, starts, pages, lens, st, cv):
        x = emb[tokens.long()]
        proj, dn = x @ w_attn.T, x @ w_dn.T
        q = spock_b200.paged_attention_prep(proj, starts, *pages, table, lens, rope=rope, q_norm=qn, k_norm=kn)
        gate = proj[:, :8 * 64].reshape(-1, 4, 2, 64)[:, :, 1]
        o = spock_b200.paged_attention(q, starts, *pages, table, lens, 0.125, gate=gate)
        qkv, z, a, b = dn.split([heads * 384, heads * 128, heads, heads], 1)
        y = spock_b200.deltanet_decode_span(layer, qkv, cv, st, a, b, z, starts)
        return torch.cat([o.reshape(-1, 256), y], 1) @ head.T, (qkv, a, b)

    state2, conv2, kp2, vp2 = state.clone(), conv.clone(), kp.clone(), vp.clone()
    length2 = length.clone()
    last = _i32([1, 2, 3])
    for rnd in range(2):
        n = [3, 1, 5]
        starts = _i32(_starts(n))
        tokens = torch.randint(0, vocab, (9,), device=DEV, generator=g).int()
        tokens[starts[:-1].long()] = last
        # plant what greedy decoding will say as the drafts, wrong from a point that differs by sequence
        for b, wrong in enumerate((1, 9, 3)):
            for i in range(1, n[b]):
                logits, _ = forward(tokens, starts, (kp.clone(), vp.clone()), length + _i32(n), state, conv)
                lo = int(starts[b])
                tokens[lo + i] = (logits[lo + i - 1].argmax() + (i == wrong)) % vocab
        length = length + _i32(n)
        logits, (qkv, a, b) = forward(tokens, starts, (kp, vp), length, state, conv)
        emitted, out = spock_b200.draft_verify(logits, tokens, starts, torch.zeros(9, device=DEV),
                                               torch.zeros(3, device=DEV), temperature=torch.zeros(3, device=DEV))
        spock_b200.deltanet_decode_span(layer, qkv, conv, state, a, b, None, starts, counts=emitted, state_out=state,
                                        conv_out=conv)
        length = length - _i32(n) + emitted
        spock_b200.Context.get(0).sync()
        assert emitted.tolist() == [1, 1, 3]
        # the same tokens one at a time
        for t in range(3):
            take = [int(t < e) for e in emitted.tolist()]
            ids = torch.cat([tokens[int(starts[i]) + t:int(starts[i]) + t + take[i]] for i in range(3)])
            one = _i32(_starts(take))
            length2 = length2 + _i32(take)
            logits1, (qkv1, a1, b1) = forward(ids, one, (kp2, vp2), length2, state2, conv2)
            spock_b200.deltanet_decode_span(layer, qkv1, conv2, state2, a1, b1, None, one, state_out=state2,
                                            conv_out=conv2)
            for i in range(3):
                if take[i]:
                    assert int(out[int(starts[i]) + t]) == int(logits1[int(one[i])].argmax())
        assert torch.equal(length, length2)
        assert torch.equal(conv, conv2)
        _check_span_state(state, state2)
        for b in range(3):
            p = torch.arange(int(length[b]), device=DEV)
            ids, slot = table[b].long()[p // page], p % page
            # the rows differ by the projection's own rounding (another batch size, another sum order): one fp16 step
            assert float((kp[ids, slot].float() - kp2[ids, slot].float()).abs().max()) <= 2 * 2.0 ** -10 * 4
            assert float((vp[ids, slot].float() - vp2[ids, slot].float()).abs().max()) <= 2 * 2.0 ** -10 * 4
        last = torch.stack([out[int(starts[b]) + int(emitted[b]) - 1] for b in range(3)])


def test_wrappers_and_binding_agree(cuda_ok):
    """The binding's short way and the wrappers' own (taken when a stream is named) give the same bits."""
    g = _gen(21)
    c = Cache([70, 9], 16, 2, 64, F16, g)
    s = _i32([0, 3, 4])
    rows = torch.randn(4, 4, 2, 64, device=DEV, generator=g).half()
    cur = torch.cuda.current_stream()
    a = spock_b200.paged_attention(rows[:, :, 0], s, *c.args(), 0.125, gate=rows[:, :, 1])
    b = spock_b200.paged_attention(rows[:, :, 0], s, *c.args(), 0.125, gate=rows[:, :, 1], stream=cur)
    assert torch.equal(a, b)
    proj = torch.randn(4, 12 * 64, device=DEV, generator=g).half()
    c2 = Cache([70, 9], 16, 2, 64, F16, _gen(21))
    a = spock_b200.paged_attention_prep(proj, s, *c.args(), rope=_table(80, 64))
    b = spock_b200.paged_attention_prep(proj, s, *c2.args(), rope=_table(80, 64), stream=cur)
    assert torch.equal(a, b) and torch.equal(c.k.view(torch.int16), c2.k.view(torch.int16))
    layer, qkv, conv, state, ga, gb, z = _span_inputs([3, 1], 4, seed=3)
    a = spock_b200.deltanet_decode_span(layer, qkv, conv, state, ga, gb, z, s)
    assert torch.equal(a, spock_b200.deltanet_decode_span(layer, qkv, conv, state, ga, gb, z, s, stream=cur))
    new = [torch.empty_like(state), torch.empty_like(conv), torch.empty_like(state), torch.empty_like(conv)]
    spock_b200.deltanet_decode_span(layer, qkv, conv, state, ga, gb, None, s, state_out=new[0], conv_out=new[1])
    spock_b200.deltanet_decode_span(layer, qkv, conv, state, ga, gb, None, s, state_out=new[2], conv_out=new[3],
                                    stream=cur)
    assert torch.equal(new[0], new[2]) and torch.equal(new[1], new[3])
    logits, tokens, ua, us, q = _verify_inputs([3, 1], 500, F16, 2, True)
    a = spock_b200.draft_verify(logits, tokens, s, ua, us, None, q)
    b = spock_b200.draft_verify(logits, tokens, s, ua, us, None, q, stream=cur)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


MORE = [
    # few rows a sequence: group sizes that do not divide the tile, a length of zero, uneven numbers of tokens
    (F16, 128, 12, 4, 16, [1] * 70, [1 + 53 * i % 900 for i in range(70)]),
    (BF16, 256, 16, 1, 16, [1, 1, 0, 1], [3000, 0, 7, 128]),
    (F16, 128, 20, 1, 16, [1, 1, 1], [77, 0, 1025]),             # 20 heads over one
    (F16, 128, 8, 2, 16, [0, 0, 1, 0], [5, 0, 40, 3]),
    (BF16, 256, 8, 2, 32, [9, 0, 0, 2, 0, 0, 0, 0, 0, 0, 0, 0], [300, 9, 0, 130] + [5] * 8),
    (F16, 128, 8, 2, 64, [1], [40000]),
    (BF16, 128, 16, 16, 16, [1] * 5, [4000, 1, 129, 128, 127]),
    # more sequences than a block has threads, many short row tiles
    (BF16, 128, 8, 4, 32, [1] * 500, [1 + 17 * i % 300 for i in range(500)]),
    (F16, 64, 4, 2, 16, [1, 0, 2] * 200, [2 + 29 * i % 200 for i in range(600)]),
    (F16, 128, 16, 4, 16, [37] * 60, [37 + 11 * i for i in range(60)]),
    (BF16, 256, 8, 2, 16, [70, 1, 5] * 14, [70 + 31 * i for i in range(42)]),
]


@pytest.mark.parametrize("case", range(len(MORE)))
def test_paged_attention_more_batches(cuda_ok, case):
    dtype, d, hq, hk, page, new, lens = MORE[case]
    g = _gen(100 + case)
    c = Cache(lens, page, hk, d, dtype, g, head_major=case % 2 == 1)
    starts, total = _starts(new), sum(new)
    q = torch.randn(total, hq, d, device=DEV, generator=g).to(dtype)
    gate = torch.randn(total, hq, d, device=DEV, generator=g).to(dtype)
    got = spock_b200.paged_attention(q, _i32(starts), *c.args(), 1 / math.sqrt(d), gate=gate)
    spock_b200.Context.get(0).sync()
    _check_attention(got, *_ref_attention(q, starts, c, 1 / math.sqrt(d), gate))


@pytest.mark.parametrize("new", [1, 7])
def test_pages_behind_the_32_bit_offsets(cuda_ok, new):
    """Pages whose elements start beyond 2^31, shared by two sequences."""
    g = _gen(8)
    pages = 2 ** 31 // (16 * 2 * 256) + 20
    c = Cache([40, 40], 16, 2, 256, F16, g)
    big = [torch.empty(pages, 16, 2, 256, dtype=F16, device=DEV) for _ in range(2)]
    far = _i32([pages - 1, pages - 9, pages - 4])
    for x, small in zip(big, (c.k, c.v)):
        x[far.long()] = small[c.table[0].long()]
    c.k, c.v = big
    c.table = far[None].repeat(2, 1).contiguous()
    starts = _starts([new, new])
    proj = torch.randn(2 * new, (8 + 4) * 256, device=DEV, generator=g).half()
    qn = torch.zeros(256, dtype=F16, device=DEV)
    q = spock_b200.paged_attention_prep(proj[:new], _i32([0, new, new]), *c.args(), q_norm=qn, k_norm=qn)
    got = spock_b200.paged_attention(torch.cat([q, q]), _i32(starts), *c.args(), 0.0625)
    spock_b200.Context.get(0).sync()
    ids, slot = c.slots(0, torch.arange(40 - new, 40, device=DEV))
    assert torch.equal(c.v[ids, slot], proj[:new, 10 * 256:].reshape(new, 2, 256))
    assert torch.equal(got[:new], got[new:])
    _check_attention(got, *_ref_attention(torch.cat([q, q]), starts, c, 0.0625, None))


def test_calls_on_two_streams_at_once(cuda_ok):
    g = _gen(9)
    jobs = []
    for lens, new in (([3000, 1500, 70], [1, 1, 1]), ([900, 2000], [5, 130])):
        c = Cache(lens, 16, 2, 256, F16, g)
        q = torch.randn(sum(new), 8, 256, device=DEV, generator=g).half()
        jobs.append((c, q, _i32(_starts(new)), torch.cuda.Stream()))
    rows = _verify_inputs([5, 3], 32003, F16, 5, True)
    starts = _i32(_starts([5, 3]))
    alone = [spock_b200.paged_attention(q, s, *c.args(), 0.0625) for c, q, s, _ in jobs]
    alone_v = spock_b200.draft_verify(*rows[:2], starts, *rows[2:4], draft_probs=rows[4])
    torch.cuda.synchronize()
    together = []
    for _ in range(10):
        for c, q, s, stream in jobs:
            with torch.cuda.stream(stream):
                together.append((spock_b200.paged_attention(q, s, *c.args(), 0.0625),
                                 spock_b200.draft_verify(*rows[:2], starts, *rows[2:4], draft_probs=rows[4])))
    torch.cuda.synchronize()
    for i, (out, verdict) in enumerate(together):
        assert torch.equal(out, alone[i % 2])
        assert all(torch.equal(x, y) for x, y in zip(verdict, alone_v))


def test_the_four_steps_captured_and_replayed(cuda_ok):
    """One graph of all four calls, replayed with other inputs, does what the calls do one by one."""
    g = _gen(12)
    new, lens, heads, vocab = [3, 1, 5], [40, 1, 300], 4, 1000
    c = Cache(lens, 16, 2, 256, F16, g)
    starts = _i32(_starts(new))
    layer, qkv, conv, state, a, b, z = _span_inputs(new, heads, seed=12)
    proj = torch.randn(9, 20 * 256, device=DEV, generator=g).half()
    rope = _table(300, 64)
    norm = torch.zeros(256, dtype=F16, device=DEV)
    logits, tokens, ua, us, _ = _verify_inputs(new, vocab, F16, 12, False)
    conv_out, state_out = torch.empty_like(conv), torch.empty_like(state)
    gates = proj[:, :16 * 256].reshape(9, 8, 2, 256)[:, :, 1]

    def step():
        q = spock_b200.paged_attention_prep(proj, starts, *c.args(), rope=rope, q_norm=norm, k_norm=norm, gated=True)
        att = spock_b200.paged_attention(q, starts, *c.args(), 0.0625, gate=gates)
        dn = spock_b200.deltanet_decode_span(layer, qkv, conv, state, a, b, z, starts)
        emitted, out = spock_b200.draft_verify(logits, tokens, starts, ua, us)
        spock_b200.deltanet_decode_span(layer, qkv, conv, state, a, b, None, starts, counts=emitted,
                                        conv_out=conv_out, state_out=state_out)
        return att, dn, emitted, out

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(3):
        proj.copy_(torch.randn(9, 20 * 256, device=DEV, generator=g))
        logits.copy_(torch.randn(9, vocab, device=DEV, generator=g) * 3)
        c.len.copy_(_i32([40 - i, 1 + i, 300 - 7 * i]))
        pages = c.k.clone(), c.v.clone()
        graph.replay()
        got = [t.clone() for t in (*held, conv_out, state_out, c.k, c.v)]
        c.k.copy_(pages[0])
        c.v.copy_(pages[1])
        want = (*step(), conv_out, state_out, c.k, c.v)
        for x, y in zip(got, want):
            assert torch.equal(x.contiguous().view(torch.uint8), y.contiguous().view(torch.uint8))
    spock_b200.Context.get(0).sync()


@pytest.mark.parametrize("probs", [False, True])
def test_draft_verify_extreme_temperatures(cuda_ok, probs):
    """Down to where only the largest logits weigh anything, up to where all weigh the same."""
    heat = [1e-42, 1e-38, 1e-30, 1e-12, 1e-6, 1e-3, 30.0, 1e6, 1e30, 3e38]
    rows = [3] * len(heat)
    logits, tokens, ua, us, q = _verify_inputs(rows, 700, BF16, 21, probs)
    logits[::3, 5:8] = logits[::3].amax(1, keepdim=True)  # several largest ones
    temp = torch.tensor(heat, device=DEV, dtype=torch.float64).float()
    assert _run_verify(logits, tokens, _starts(rows), ua, us, temp, q) == \
        _ref_verify(logits, tokens, _starts(rows), ua, us, temp, q)


def test_draft_verify_many_sequences(cuda_ok):
    rows = [1 + i % 3 for i in range(700)]
    logits, tokens, ua, us, q = _verify_inputs(rows, 130, F16, 22, True)
    assert _run_verify(logits, tokens, _starts(rows), ua, us, None, q) == \
        _ref_verify(logits, tokens, _starts(rows), ua, us, None, q)


def test_paged_attention_refuses_scales_and_strides(cuda_ok):
    g = _gen(1)
    c = Cache([20], 16, 2, 64, F16, g)
    q = torch.randn(2, 8, 64, device=DEV, generator=g).half()
    call = lambda q, scale: spock_b200.paged_attention(q, _i32([0, q.shape[0]]), *c.args(), scale)
    for scale in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(spock_b200.SpockError, match="positive and finite"):
            call(q, scale)
    for bad in (q[:1].expand(2, -1, -1), q[:, :1].expand(-1, 8, -1)):
        with pytest.raises(spock_b200.SpockError, match="strides must be positive"):
            call(bad, 1.0)
    # a stride that is never used may be anything
    one = torch.as_strided(q, (1, 8, 64), (0, 64, 1))
    assert torch.equal(call(one, 1.0), call(q[:1], 1.0))


@pytest.mark.parametrize("dtype,d,hq,hk,new,lens", [
    (F16, 256, 8, 2, [60] * 3, [4575] * 3),     # row tiles of full rows in a dozen parts each
    (BF16, 128, 16, 2, [40], [60000]),          # in some hundred
    (F16, 256, 16, 1, [1, 1], [30000, 20000]),  # few rows, some seventy parts
    (BF16, 64, 4, 4, [200], [12000]),
])
def test_paged_attention_row_tiles_in_many_parts(cuda_ok, dtype, d, hq, hk, new, lens):
    g = _gen(31)
    c = Cache(lens, 64, hk, d, dtype, g)
    starts = _starts(new)
    q = torch.randn(sum(new), hq, d, device=DEV, generator=g).to(dtype)
    gate = torch.randn(sum(new), hq, d, device=DEV, generator=g).to(dtype)
    got = spock_b200.paged_attention(q, _i32(starts), *c.args(), 1 / math.sqrt(d), gate=gate)
    spock_b200.Context.get(0).sync()
    _check_attention(got, *_ref_attention(q, starts, c, 1 / math.sqrt(d), gate))
