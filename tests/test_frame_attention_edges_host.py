"""Frame attention without a GPU: what the layer books, and which overlaps of operands are refused."""
import pytest
import torch


# ---- the layer's state ----

def test_a_replaced_state_leaves_the_list_of_caches():
    """Alternating numbers of streams: the caches of one state at a time are booked, beside other layers' buffers."""
    from deltacnn_amd.sparse_layers import DCFrameAttention, DCModule
    saved, DCModule.temp_buffers = DCModule.temp_buffers, []
    try:
        other = DCModule._cache(torch.zeros(5))
        layer = DCFrameAttention(16, 2, frames=2, page_size=8)
        sizes = []
        for b in (1, 2, 1, 2, 1):
            layer._drop()
            layer._state = layer._start(torch.zeros(b, 16, 3, 3))
            sizes.append(DCModule.get_temp_buffer_numel() - other.numel())
        assert sizes[0] > 0 and sizes == [sizes[0] * b for b in (1, 2, 1, 2, 1)]
        assert DCModule.temp_buffers[0] is other
        layer._captured.append(layer._state)  # a graph goes on with this one
        layer._drop()
        assert DCModule.get_temp_buffer_numel() - other.numel() == sizes[0]
        layer.reset()
        assert DCModule.get_temp_buffer_numel() == 0 and layer._captured == []
    finally:
        DCModule.temp_buffers = saved
