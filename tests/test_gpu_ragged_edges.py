"""Values and calls at the edges of the ragged steps."""
import pytest
import torch

import spock_b200
from tests.test_gpu_ragged import DEV, F16, _i32, _span_inputs

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
