"""The attention of beams as the first call on a device, inside a capture."""
import pytest
import torch

from test_gpu_beams import K, _attention, _beams, _near  # noqa: F401

pytestmark = pytest.mark.gpu


def test_a_first_call_inside_a_capture_is_refused(K, monkeypatch):  # noqa: F811
    """The device's error word (and the counters that the products share) would be cleared by the graph's replays alone, and hold anything ahead of
    the first.  A call in front of the capture makes them."""
    from rustinfer_b200.ops.library import KernelError
    q, cache, table, kv_len, sh = _beams(2, 2, 4, 2, 64, 16, [90, 70], [[9, 3], [1, 20]], seed=4)
    table, out, other = table.clamp(min=0), torch.empty_like(q), torch.zeros(8, device="cuda")
    monkeypatch.setattr(K, "_tc_state", {})                # as on a device nobody has used

    def call():
        K.attention_decode_beams(q, out, cache, table, kv_len, sh, 2, 4, 2, 64, 0.125, None, 90, 20)
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        other.add_(1)
        with pytest.raises(KernelError, match="capture"):
            call()
        assert not K._tc_state
    call()
    assert K.gemm_tc_error(q.device) == 0
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    out.zero_()
    graph.replay()
    _near(out, *_attention(q, cache, table, kv_len, 4, 2, 64, 0.125, None), 64, 110)
