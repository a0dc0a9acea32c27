"""The ragged steps' checks of their arguments that need no GPU: the C entry
points without a context, and the Python wrappers' types, shapes and devices."""
import ctypes

import pytest
import torch

import spock_b200

F16, F32, I32 = torch.float16, torch.float32, torch.int32


def test_null_context_is_rejected():
    L = spock_b200.lib()
    kv, layer, n = spock_b200.PagedKv(), spock_b200.DnLayer(), ctypes.c_size_t()
    calls = {
        "spock_paged_attention_prep": lambda: L.spock_paged_attention_prep(
            None, ctypes.byref(kv), 1, None, 0, None, 0, 1, 0, None, None, 1e-6, None, 0, 0, None, None),
        "spock_paged_attention": lambda: L.spock_paged_attention(
            None, ctypes.byref(kv), 1, None, 0, 1, None, 0, 0, None, 0, 0, 1.0, None, None, 0, None),
        "spock_paged_attention_workspace": lambda: L.spock_paged_attention_workspace(None, 1, 1, 64, ctypes.byref(n)),
        "spock_deltanet_decode_span": lambda: L.spock_deltanet_decode_span(
            None, ctypes.byref(layer), 1, None, None, 0, None, 0, None, None, 0, None, 0, *([None] * 6)),
        "spock_draft_verify": lambda: L.spock_draft_verify(
            None, 0, None, 0, 0, 1, 1, None, None, None, 0, *([None] * 6), 0, None),
        "spock_draft_verify_workspace": lambda: L.spock_draft_verify_workspace(None, 1, 1, 1, ctypes.byref(n)),
    }
    for name, call in calls.items():
        assert call() == spock_b200.SPOCK_ERR_INVALID, name
        assert name.encode() in L.spock_last_error(None)


def _attn(**change):
    a = dict(q=torch.zeros(3, 8, 64, dtype=F16), start=torch.tensor([0, 3], dtype=I32),
             k_pages=torch.zeros(2, 16, 2, 64, dtype=F16), v_pages=torch.zeros(2, 16, 2, 64, dtype=F16),
             page_table=torch.zeros(1, 2, dtype=I32), kv_len=torch.tensor([3], dtype=I32), scale=1.0)
    a.update(change)
    return spock_b200.paged_attention(**a)


@pytest.mark.parametrize("change,text", [
    ({}, "CUDA"),
    ({"q": torch.zeros(3, 8, 64)}, "q: expected torch.float16"),
    ({"q": torch.zeros(3, 512, dtype=F16)}, "q: expected 3 dimensions"),
    ({"q": torch.zeros(3, 8, 128, dtype=F16)[..., ::2]}, "contiguous last dimension"),
    ({"start": torch.tensor([0, 3])}, "start: expected torch.int32"),
    ({"kv_len": torch.zeros(4, dtype=I32)[::2]}, "kv_len: expected a contiguous tensor"),
    ({"v_pages": torch.zeros(2, 16, 2, 64)}, "v_pages: expected torch.float16"),
    ({"gate": torch.zeros(3, 8, 64)}, "gate: expected torch.float16"),
    ({"out": torch.zeros(64, 8, 3, dtype=F16).permute(2, 1, 0)}, "out: expected a contiguous tensor"),
])
def test_paged_attention_rejects(change, text):
    with pytest.raises(spock_b200.SpockError, match=text) as e:
        _attn(**change)
    assert e.value.code == spock_b200.SPOCK_ERR_INVALID


def test_draft_verify_rejects():
    x = torch.zeros(2, 10, dtype=F16)
    one = torch.zeros(2, dtype=F32)
    with pytest.raises(spock_b200.SpockError, match="tokens: expected torch.int32"):
        spock_b200.draft_verify(x, torch.zeros(2), torch.tensor([0, 2], dtype=I32), one, one[:1])
    with pytest.raises(spock_b200.SpockError, match="fp32, fp16 or bf16") as e:
        spock_b200.draft_verify(x.double(), torch.zeros(2, dtype=I32), torch.tensor([0, 2], dtype=I32), one, one[:1])
    assert e.value.code == spock_b200.SPOCK_ERR_UNSUPPORTED


def test_deltanet_decode_span_rejects():
    layer = spock_b200.DeltaNetLayer(torch.zeros(768, 4, dtype=F16), torch.zeros(2, 2), torch.zeros(128), num_heads=2)
    half = lambda *s: torch.zeros(*s, dtype=F16)
    with pytest.raises(spock_b200.SpockError, match="state: expected torch.float32"):
        spock_b200.deltanet_decode_span(layer, half(1, 768), half(1, 768, 4), half(1, 2, 128, 128), half(1, 2),
                                        half(1, 2), half(1, 256), torch.tensor([0, 1], dtype=I32))
