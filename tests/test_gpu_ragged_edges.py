"""Values and calls at the edges of the ragged steps: scores of any size, NaN and
infinities in queries, weights far below a row's largest, group sizes that leave
pad rows, tensors at odd offsets, outputs over inputs, named streams."""
import math

import pytest
import torch

import spock_b200
from tests.test_gpu_ragged import (BF16, DEV, F16, Cache, _check_attention, _gen, _half_step, _i32, _ref_attention,
                                   _ref_verify, _run_verify, _span_inputs, _starts, _verify_inputs)

pytestmark = pytest.mark.gpu


def _at_offset(t, n):
    """The same values n elements behind a 256-byte boundary."""
    return torch.cat([t.new_zeros(n), t.flatten()])[n:].view(t.shape)


def test_deltanet_decode_span_at_odd_offsets(cuda_ok):
    """Weights and rows anywhere their type allows give the same bits; where wide accesses need more, the call is
    refused before it launches anything."""
    layer, qkv, conv, state, a, b, z = _span_inputs([3, 2], 4, seed=1)
    s = _i32([0, 3, 5])
    span = spock_b200.deltanet_decode_span
    want = span(layer, qkv, conv, state, a, b, z, s)
    for n in (1, 2, 3):
        odd = spock_b200.DeltaNetLayer(layer.conv_weight, _at_offset(layer.a_log_bias, n),
                                       _at_offset(layer.norm_weight, n), num_heads=4)
        got = span(odd, _at_offset(qkv, n), conv, state, _at_offset(a, n), _at_offset(b, n), _at_offset(z, n), s)
        assert torch.equal(got, want)
    outs = torch.zeros(5 * 512 + 4, dtype=F16, device=DEV)
    assert torch.equal(span(layer, qkv, conv, state, a, b, z, s, out=outs[4:].view(5, 512)), want)
    for stream in (None, torch.cuda.current_stream()):
        for n in (1, 2, 3):
            with pytest.raises(spock_b200.SpockError, match="out 8-byte") as e:
                span(layer, qkv, conv, state, a, b, z, s, out=outs[n:n + 2560].view(5, 512), stream=stream)
            assert e.value.code == spock_b200.SPOCK_ERR_INVALID
        for change in (dict(conv_state=_at_offset(conv, 1)), dict(state=_at_offset(state, 2))):
            args = dict(conv_state=conv, state=state)
            args.update(change)
            with pytest.raises(spock_b200.SpockError, match="aligned") as e:
                span(layer, qkv, args["conv_state"], args["state"], a, b, z, s, stream=stream)
            assert e.value.code == spock_b200.SPOCK_ERR_INVALID


# dtype, head_dim, q_heads, kv_heads, new tokens, lengths: both kernels, row tiles of one CTA and of several
KERNELS = [
    (F16, 128, 8, 2, [1, 1], [100, 40]),
    (BF16, 256, 8, 2, [1], [40000]),
    (F16, 128, 6, 2, [1, 1], [30000, 700]),
    (BF16, 128, 8, 2, [5, 9], [100, 40]),
    (F16, 256, 8, 2, [40], [9000]),
    (BF16, 64, 4, 2, [3, 1], [5000, 4]),
    # the kernel for few rows: 64 sequences and more, no more tokens than those, head size 256, groups up to 4
    (F16, 256, 8, 2, [1] * 70, [100 - i for i in range(70)]),
    (BF16, 256, 8, 2, [1, 1] + [0] * 70, [40000, 77] + [0] * 70),
    (F16, 256, 6, 2, [1, 0, 1] + [0] * 70, [30000, 5, 700] + [0] * 70),
    (BF16, 256, 4, 4, [3, 1, 40] + [0] * 70, [5000, 4, 1700] + [0] * 70),
]


def _case(case, seed):
    dtype, d, hq, hk, new, lens = KERNELS[case]
    g = _gen(seed + case)
    c = Cache(lens, 16, hk, d, dtype, g)
    q = torch.randn(sum(new), hq, d, device=DEV, generator=g).to(dtype)
    return c, q, _starts(new)


def _attend(q, starts, c, scale):
    got = spock_b200.paged_attention(q, _i32(starts), *c.args(), scale)
    spock_b200.Context.get(0).sync()
    return got


@pytest.mark.parametrize("case", range(len(KERNELS)))
def test_equal_scores_average_the_values(cuda_ok, case):
    """All of a row's scores equal, from -2^100 (what the type holds of it) to 2^30: every weight is the same."""
    c, q, starts = _case(case, 200)
    big = 2.0 ** 50 if c.k.dtype == BF16 else 2.0 ** 15
    for a, b in ((0.0, 1.0), (2.0 ** 15, 2.0 ** 15), (big, -big), (-(2.0 ** 13) * 1.25, 1.125 * 2.0 ** 14)):
        q.zero_()
        q[..., 5], c.k[..., 5] = a, b
        for other in (0, 17):  # more than one product to a score
            c.k[..., other] = 0.0
        got = _attend(q, starts, c, 1.0)
        # every term of a score but one is exactly 0, so the scores are exact and equal
        ref, mag, _ = _ref_attention(q, starts, c, 1.0, None)
        _check_attention(got, ref, mag, torch.zeros_like(mag))


@pytest.mark.parametrize("case", range(len(KERNELS)))
def test_nan_and_infinite_queries_stay_in_their_rows(cuda_ok, case):
    """A row whose query holds NaN, or whose scores are all -inf, is NaN, whole or in parts; all others are as ever."""
    c, q, starts = _case(case, 210)
    c.k[..., 0] = -c.k[..., 0].abs() - 0.5
    ref, mag, err = _ref_attention(q, starts, c, 0.125, None)
    nan = torch.zeros(q.shape[:2], dtype=torch.bool, device=DEV)
    for i, value in enumerate((math.nan, math.inf)):
        t, h = i * (q.shape[0] - 1), i * 3
        q[t, h] = 0.0
        q[t, h, 0] = value  # +inf times negative keys, and zeros: every score -inf
        nan[t, h] = True
    got = _attend(q, starts, c, 0.125)
    assert bool(torch.isnan(got[nan]).all())
    _check_attention(got[~nan], ref[~nan], mag[~nan], err[~nan])


@pytest.mark.parametrize("dtype,d,n,length", [(F16, 128, 152, 150), (BF16, 256, 300, 290), (F16, 64, 7, 4)])
def test_nan_queries_that_see_nothing(cuda_ok, dtype, d, n, length):
    """Tokens before position 0 are zero whatever their queries hold, also beside tokens that see several tiles."""
    g = _gen(5)
    c = Cache([length], 16, 2, d, dtype, g)
    q = torch.randn(n, 8, d, device=DEV, generator=g).to(dtype)
    q[0, 1], q[1, 2, 3] = math.nan, math.inf
    got = _attend(q, [0, n], c, 0.125)
    blind = n - length
    assert bool((got[:blind] == 0).all())
    q[:2] = 0
    ref = _ref_attention(q, [0, n], c, 0.125, None)
    _check_attention(got[blind:], *(t[blind:] for t in ref))


@pytest.mark.parametrize("case", range(len(KERNELS)))
def test_equal_scores_that_do_not_round_to_powers(cuda_ok, case):
    """Equal scores of some 2^32, whose product with log2(e) fp32 does not hold: still the average of the values."""
    c, q, starts = _case(case, 240)
    for a, b in ((57344.0, 61440.0), (61440.0, 63488.0), (-57344.0, 61440.0)):
        q.zero_()
        q[..., 5], c.k[..., 5] = a, b
        got = _attend(q, starts, c, 1.0)
        ref, mag, _ = _ref_attention(q, starts, c, 1.0, None)
        _check_attention(got, ref, mag, torch.zeros_like(mag))


def _decode_us(group, d=256, seqs=256):
    g = _gen(7)
    lens = [65 + 13 * i % 1086 for i in range(seqs)]
    c = Cache(lens, 64, 2, d, F16, g)
    q = torch.randn(seqs, 2 * group, d, device=DEV, generator=g).half()
    s = _i32(_starts([1] * seqs))
    run = lambda: spock_b200.paged_attention(q, s, *c.args(), 0.0625)
    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()  # noqa: F841
    times = []
    for _ in range(30):
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        graph.replay()
        b.record()
        b.synchronize()
        times.append(a.elapsed_time(b) * 1e3)
    return sorted(times)[15]


@pytest.mark.parametrize("group", [1, 2, 3, 5, 6, 7])
def test_pad_rows_cost_nothing(cuda_ok, group):
    """Decode reads the cache whatever the group size: one that leaves pad rows is no slower than the next one of 4."""
    seen = []
    for _ in range(3):  # another job's moment on the machine may fall into one of them
        seen.append((_decode_us(group), _decode_us((group + 3) // 4 * 4)))
        if seen[-1][0] <= 1.1 * seen[-1][1]:
            return
    pytest.fail(f"us of this group and of the full one: {seen}")


@pytest.mark.parametrize("case", range(len(KERNELS)))
def test_weights_far_below_the_largest(cuda_ok, case):
    """One position in 64 weighs e^16 times as much as the others, whose values are all that is seen."""
    c, q, starts = _case(case, 220)
    for b, n in enumerate(c.lens):
        p = torch.arange(n, device=DEV)
        ids, slot = c.slots(b, p)
        c.k[ids, slot] = 0.0
        c.v[ids, slot] = 1000.0
        few = p % 64 == 0
        c.k[ids[few], slot[few], :, 3] = 16.0
        c.v[ids[few], slot[few]] = 0.0
    q.zero_()
    q[..., 3] = 1.0
    got = _attend(q, starts, c, 1.0).double()
    ref, mag, _ = _ref_attention(q, starts, c, 1.0, None)
    # as in _check_attention, with exact scores; and fp16 weights, kept with 7 more octaves below the row's
    # largest than fp16's own 2^-24: off by 2^-32 of it each, 63 of 64 positions 1000 times that
    e = _half_step(q.dtype)
    tol = e * ref.abs() + (2 * e + 2.0 ** -15) * mag
    if q.dtype == F16:
        tol = tol + 6e-8 + 64 * 1000 * 2.0 ** -32
    off = (got - ref).abs()
    assert bool((off <= tol).all()), float((off / tol).max())


@pytest.mark.parametrize("case", range(len(KERNELS)))
def test_weights_sum_to_one(cuda_ok, case):
    """Values that are all the same come out as they are (times the gate), whatever the weights' roundings."""
    c, q, starts = _case(case, 230)
    c.k *= 4  # some weights carry most of a row, in tiles behind the first
    c.v[:] = torch.where(torch.isnan(c.v), math.nan, 1.0)
    gate = torch.randn(q.shape, device=DEV, generator=_gen(case)).to(q.dtype)
    got = spock_b200.paged_attention(q, _i32(starts), *c.args(), 0.125, gate=gate)
    spock_b200.Context.get(0).sync()
    ref = torch.sigmoid(gate.double())
    # the output's rounding; both sums of weights in fp32, in chains of at most 2^9 steps of 2^-23 (the matrix
    # instructions may cut off what they add); 2^-15 for the division and the gate. No rounding of weights.
    tol = (_half_step(q.dtype) + 2 * 2.0 ** -14 + 2.0 ** -15) * ref
    off = (got.double() - ref).abs()
    assert bool((off <= tol).all()), float((off / tol).max())


def test_draft_verify_refuses_outputs_over_its_inputs(cuda_ok):
    """Threads that write out_tokens would race with those that still read tokens: refused on the host."""
    logits, tokens, ua, us, _ = _verify_inputs([3, 2], 50, F16, 3, False)
    buf = torch.zeros(16, dtype=torch.int32, device=DEV)
    buf[:3], buf[3:8] = _i32([0, 3, 5]), tokens
    start, toks = buf[:3], buf[3:8]
    want = spock_b200.draft_verify(logits, tokens, _i32([0, 3, 5]), ua, us)
    for stream in (None, torch.cuda.current_stream()):
        call = lambda **k: spock_b200.draft_verify(logits, toks, start, ua, us, stream=stream, **k)
        for bad in (dict(out_tokens=toks), dict(out_tokens=buf[7:12]), dict(out_tokens=buf[2:7]),
                    dict(emitted=buf[7:9]), dict(emitted=buf[1:3]), dict(out_tokens=buf[8:13], emitted=buf[12:14])):
            with pytest.raises(spock_b200.SpockError, match="must not overlap") as e:
                call(**bad)
            assert e.value.code == spock_b200.SPOCK_ERR_INVALID
        got = call(out_tokens=buf[8:13], emitted=buf[13:15])  # side by side is apart
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        assert torch.equal(toks, tokens)


def test_deltanet_decode_span_refuses_shifted_states(cuda_ok):
    """New states over another sequence's old ones would race with their reads; in place and apart are fine."""
    layer, qkv, conv, state, a, b, z = _span_inputs([2, 1], 4, seed=1)
    s = _i32([0, 2, 3])
    pool, pool_c = torch.zeros(5, *state.shape[1:], device=DEV), torch.zeros(5, *conv.shape[1:], dtype=F16, device=DEV)
    pool[1:3], pool_c[1:3] = state, conv
    run = lambda st, cv, **k: spock_b200.deltanet_decode_span(layer, qkv, pool_c[1:3], pool[1:3], a, b, None, s,
                                                              state_out=st, conv_out=cv, **k)
    for stream in (None, torch.cuda.current_stream()):
        for i, j in ((0, 1), (2, 1), (1, 2), (1, 0), (0, 3), (3, 2)):
            with pytest.raises(spock_b200.SpockError, match="apart from them") as e:
                run(pool[i:i + 2], pool_c[j:j + 2], stream=stream)
            assert e.value.code == spock_b200.SPOCK_ERR_INVALID
    run(pool[3:5], pool_c[3:5])
    run(pool[1:3], pool_c[1:3])
    spock_b200.Context.get(0).sync()
    assert torch.equal(pool[1:3], pool[3:5]) and torch.equal(pool_c[1:3], pool_c[3:5])


def test_named_streams_do_not_take_memory_in_use(cuda_ok):
    """Memory that the current stream has freed, with work on it still queued, is not what a call on another stream
    gets for its outputs and workspaces."""
    g = _gen(6)
    c, starts = Cache([900, 130], 16, 2, 256, F16, g), _i32([0, 200, 300])
    q = torch.randn(300, 8, 256, device=DEV, generator=g).half()
    proj = torch.randn(300, 20 * 256, device=DEV, generator=g).half()
    layer, qkv, conv, state, a, b, z = _span_inputs([200, 100], 4, seed=1)
    logits, tokens, ua, us, _ = _verify_inputs([200, 100], 5000, F16, 3, False)
    side = torch.cuda.Stream()
    calls = [lambda **k: (spock_b200.paged_attention(q, starts, *c.args(), 0.0625, **k),),
             lambda **k: (spock_b200.paged_attention_prep(proj, starts, *c.args(), **k),),
             lambda **k: (spock_b200.deltanet_decode_span(layer, qkv, conv, state, a, b, z, starts, **k),),
             lambda **k: spock_b200.draft_verify(logits, tokens, starts, ua, us, **k)]
    for call in calls:
        want = [t.clone() for t in call()]
        torch.cuda.synchronize()
        sizes = [t.numel() * t.element_size() for t in want] + [1 << 25, 1 << 23, 1 << 21, 1 << 12]
        held = [torch.empty(n, dtype=torch.uint8, device=DEV) for n in sizes for _ in range(2)]
        was = {t.data_ptr() for t in held}
        torch.cuda._sleep(40_000_000)  # some 20 ms
        for t in held:
            t.fill_(255)
        del held, t
        got = call(stream=side)
        assert not was & {t.data_ptr() for t in got}
        side.synchronize()
        torch.cuda.synchronize()
        for x, y in zip(got, want):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


@pytest.mark.parametrize("case", range(len(KERNELS)))
def test_scales_that_take_scores_out_of_range(cuda_ok, case):
    """Scaled scores that fp32 does not hold: a row is its largest score's value (or the average of equal ones)."""
    c, q, starts = _case(case, 250)
    c.k.copy_(torch.where(torch.isnan(c.k), math.nan, torch.round(c.k * 2)))
    q.copy_(torch.round(q))  # whole numbers: scores are exact, the largest ones are equal or at least 1 apart
    q[..., 16:] = 0
    got = _attend(q, starts, c, 2.0 ** 125)
    ref, mag, _ = _ref_attention(q, starts, c, 2.0 ** 125, None)
    _check_attention(got, ref, mag, torch.zeros_like(mag))


@pytest.mark.parametrize("case", range(len(KERNELS)))
def test_scales_next_to_zero(cuda_ok, case):
    """The smallest normal scale and subnormal ones: all positions weigh the same."""
    c, q, starts = _case(case, 260)
    for scale in (2.0 ** -126, 2.0 ** -140, 2.0 ** -149):
        got = _attend(q, starts, c, scale)
        _check_attention(got, *_ref_attention(q, starts, c, scale, None))


def test_scales_that_overflow_with_log2e_are_refused(cuda_ok):
    """The kernels work with scale * log2(e): one that makes that infinite would turn every row into NaN."""
    c, q, starts = _case(0, 270)
    top = torch.finfo(torch.float32).max
    for scale in (top, top / 1.44, 2.4e38):
        with pytest.raises(spock_b200.SpockError, match="positive and finite") as e:
            _attend(q, starts, c, scale)
        assert e.value.code == spock_b200.SPOCK_ERR_INVALID
    assert not bool(torch.isnan(_attend(q, starts, c, top / 1.4427)).any())


def test_draft_verify_at_subnormal_temperatures(cuda_ok):
    """Logits and temperatures so small that log2(e) / T is not an fp32 number: 64 bits still tell the logits apart."""
    rows, vocab = [2] * 8, 1000
    logits = -torch.arange(vocab, device=DEV).repeat(16, 1).float() * 2.0 ** -149
    tokens = torch.tensor([0, 5] * 8, dtype=torch.int32, device=DEV)
    ua = torch.linspace(0.0, 0.01, 16, device=DEV)
    us = torch.linspace(0.0, 0.99, 8, device=DEV)
    temp = torch.tensor([2.0 ** -140, 2.0 ** -149] * 4, device=DEV)
    starts = _starts(rows)
    got = _run_verify(logits, tokens, starts, ua, us, temp, None)
    assert got == _ref_verify(logits, tokens, starts, ua, us, temp, None)


@pytest.mark.parametrize("group", [1, 2, 3, 4])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_batches_of_few_rows(cuda_ok, group, dtype):
    """The kernel for decode batches: lengths of zero and one, ends on and beside a tile's border, sequences with
    nothing and with several tokens among them, pages either way round, gates; the same bits every time."""
    g = _gen(300 + group)
    new = [1] * 90 + [0, 5, 0, 0, 17, 0, 0, 0, 2, 0, 0, 0] + [0] * 30
    lens = ([0, 1, 2, 127, 128, 129, 130, 255, 256, 257, 4000] * 9)[:90] + [7, 3, 0, 200, 300, 1, 1, 128, 2, 0, 5, 9] + [3] * 30
    c = Cache(lens, 16 if group % 2 else 24, 2, 256, dtype, g, head_major=group > 2)
    starts, total = _starts(new), sum(new)
    rows = torch.randn(total + 2, 2 * group, 2, 256, device=DEV, generator=g).to(dtype)
    q, gate = rows[:, :, 0], rows[:, :, 1]
    out = torch.full((total + 2, 2 * group, 256), 7.0, dtype=dtype, device=DEV)
    assert total + 2 <= len(new)
    spock_b200.paged_attention(q, _i32(starts), *c.args(), 0.0625, gate=gate, out=out)
    spock_b200.Context.get(0).sync()
    assert bool((out[total:] == 7.0).all())
    ref = _ref_attention(q, starts, c, 0.0625, gate)
    _check_attention(out[:total], *(t[:total] for t in ref))
    for _ in range(3):
        assert torch.equal(spock_b200.paged_attention(q, _i32(starts), *c.args(), 0.0625, gate=gate)[:total], out[:total])


def test_nan_queries_of_few_rows_that_see_nothing(cuda_ok):
    g = _gen(5)
    c = Cache([7] + [1] * 70, 16, 2, 256, F16, g)
    q = torch.randn(10, 8, 256, device=DEV, generator=g).half()
    q[0, 1], q[1, 2, 3] = math.nan, math.inf
    got = _attend(q, _starts([10] + [0] * 70), c, 0.0625)
    assert bool((got[:3] == 0).all())
    q[:2] = 0
    ref = _ref_attention(q, _starts([10] + [0] * 70), c, 0.0625, None)
    _check_attention(got[3:], *(t[3:] for t in ref))


def test_tables_whose_last_tile_passes_31_bits_are_refused(cuda_ok):
    pages = torch.zeros(1, 114808, 1, 64, dtype=F16, device=DEV)
    table = torch.zeros(1, 18705, dtype=torch.int32, device=DEV)  # 2^31 - 8 positions
    q, proj = torch.zeros(1, 4, 64, dtype=F16, device=DEV), torch.zeros(1, 6 * 64, dtype=F16, device=DEV)
    one, s = _i32([1]), _i32([0, 1])
    for call in (lambda t: spock_b200.paged_attention(q, s, pages, pages, t, one, 1.0),
                 lambda t: spock_b200.paged_attention_prep(proj, s, pages, pages.clone(), t, one, gated=False)):
        with pytest.raises(spock_b200.SpockError, match="positions per sequence") as e:
            call(table)
        assert e.value.code == spock_b200.SPOCK_ERR_UNSUPPORTED
        call(table[:, :18704])
        spock_b200.Context.get(0).sync()


def test_named_streams_captured(cuda_ok):
    """Calls on a stream that joined a capture: their memory is the graph's, and replays give the calls' bits."""
    g = _gen(8)
    c, starts = Cache([900, 130], 16, 2, 256, F16, g), _i32([0, 5, 12])
    q = torch.randn(12, 8, 256, device=DEV, generator=g).half()
    layer, qkv, conv, state, a, b, z = _span_inputs([5, 7], 4, seed=1)
    logits, tokens, ua, us, _ = _verify_inputs([5, 7], 5000, F16, 3, False)
    side = torch.cuda.Stream()

    def step(stream):
        return (spock_b200.paged_attention(q, starts, *c.args(), 0.0625, stream=stream),
                spock_b200.deltanet_decode_span(layer, qkv, conv, state, a, b, z, starts, stream=stream),
                *spock_b200.draft_verify(logits, tokens, starts, ua, us, stream=stream))

    want = [t.clone() for t in step(None)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        side.wait_stream(torch.cuda.current_stream())
        held = step(side)
        torch.cuda.current_stream().wait_stream(side)
    for _ in range(2):
        others = [torch.full((1 << n,), 255, dtype=torch.uint8, device=DEV) for n in (12, 16, 20, 25)]
        graph.replay()
        torch.cuda.synchronize()
        assert all(bool((t == 255).all()) for t in others)
        for x, y in zip(held, want):
            assert torch.equal(x, y)
