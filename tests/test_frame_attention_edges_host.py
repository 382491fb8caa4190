"""Frame attention without a GPU: what the layer books, and which overlaps of operands are refused."""
import random

import pytest
import torch

from test_frame_attention_host import attention_args, rotary_args


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


@pytest.mark.parametrize("change", [dict(head_dim=264), dict(head_dim=12), dict(sections=(3, 5, 8)), dict(sections=(-2, 8, 8)),
                                    dict(sections=(8, 8)), dict(sections=(0, 0, 0)), dict(kv_heads=3), dict(frames=0), dict(keep_frames=-1),
                                    dict(page_size=0)], ids=str)
def test_the_layer_refuses_what_its_operators_refuse(change):
    from deltacnn_amd.sparse_layers import DCFrameAttention
    with pytest.raises(ValueError, match="DCFrameAttention"):
        DCFrameAttention(64, 4, **change)


# ---- rows that share a buffer ----

BASE = 1 << 20  # addresses that are compared and never read: every call here is refused before it would launch


def rows(dims, column=0):
    """(offset, token stride, head stride) of rows in a dense buffer: `dims` names its dimensions, (size, "t" | "h" | "x"),
    from the outermost; "x" are those in which `column` counts."""
    stride, out = 1, {"t": None, "h": None, "x": 0}
    for size, what in reversed(dims):
        if what == "x":
            out["x"] += column % size * stride
            column //= size
        elif what != "d":
            out[what] = stride
        stride *= size
    return out["x"], out["t"], out["h"]


def append_verdict(lib, tokens, q_heads, kv_heads, dim, q, out, k, v):
    """What dc_rotary says of rows (offset, token stride, head stride): its message.  The cache, far away, has its keys
    over its values, which is refused behind the rows."""
    at = lambda r: BASE + 2 * r[0]  # noqa: E731
    a = rotary_args(BASE, tokens=tokens, q_heads=q_heads, kv_heads=kv_heads, dim=dim, sections=(dim, 0, 0, 0), axes=1,
                    q=at(q), q_token_stride=q[1], q_head_stride=q[2], out=at(out), out_token_stride=out[1], out_head_stride=out[2],
                    k=at(k), k_token_stride=k[1], k_head_stride=k[2], v=at(v), v_token_stride=v[1], v_head_stride=v[2],
                    streams=1, keys=BASE + (1 << 24), values=BASE + (1 << 24), weights=None, stamps=None)
    assert lib.dc_rotary(a, 1, None) == -3 and lib.dc_last_kernels() == b""
    return lib.dc_last_error().decode()


@pytest.mark.parametrize("tokens", [1, 2, 5])
@pytest.mark.parametrize("heads", [1, 2, 3])
def test_columns_of_one_projection_are_apart(lib, tokens, heads):
    """q, k and v in one buffer, whatever the order of its dimensions, and out in place of q."""
    dim, t, h, x, d = 16, (tokens, "t"), (heads, "h"), (3, "x"), (16, "d")
    for dims in ((t, x, h, d), (t, h, x, d), (h, t, x, d), (h, x, t, d), (x, t, h, d), (x, h, t, d)):
        q, k, v = (rows(dims, c) for c in range(3))
        said = append_verdict(lib, tokens, heads, heads, dim, q, q, k, v)
        assert "keys and values overlap" in said, (dims, said)
        # one element further and they are not
        said = append_verdict(lib, tokens, heads, heads, dim, (q[0] + 1, *q[1:]), (q[0] + 1, *q[1:]), k, v)
        assert "out overlaps k or v" in said, (dims, said)
    # fewer kv heads, behind the query heads of a token
    q, k, v = (0, (heads + 2) * dim, dim), (heads * dim, (heads + 2) * dim, dim), ((heads + 1) * dim, (heads + 2) * dim, dim)
    assert "keys and values overlap" in append_verdict(lib, tokens, heads, 1, dim, q, q, k, v)


def test_rows_that_share_an_element_are_never_taken_for_apart(lib):
    rng, verdicts = random.Random(7), []
    for _ in range(3000):
        dim, sets = rng.choice([4, 8]), []
        tokens = rng.randint(1, 4)
        for heads in (rng.randint(1, 4), rng.randint(1, 4)):
            inner = rng.choice([dim, dim + 4, 2 * dim, 3 * dim, 5 * dim])
            n = rng.choice([tokens, heads])
            outer = inner * rng.choice([n, n, n + 1, 2 * n, 3 * n])
            ts, hs = (inner, outer) if n == tokens and rng.random() < 0.7 else (outer, inner)
            sets.append((rng.randint(0, 12) * 4, ts, hs, heads))
        (*out, qh), (*k, kh) = sets
        used = [{r[0] + t * r[1] + g * r[2] + e for t in range(tokens) for g in range(n) for e in range(dim)} for r, n in ((out, qh), (k, kh))]
        said = append_verdict(lib, tokens, qh, kh, dim, out, out, k, (1 << 18, kh * dim, dim))
        if "overlap each other" in said:  # rows of out among themselves
            continue
        shared = bool(used[0] & used[1])
        verdicts.append((shared, "out overlaps k or v" in said))
        assert not shared or verdicts[-1][1], (tokens, dim, sets, said)
    # the other way round a few layouts are refused that would do: none of those above, and not many
    assert sum(s for s, _ in verdicts) > 300 and sum(not s for s, _ in verdicts) > 300
    assert sum(r for s, r in verdicts if not s) < 0.2 * sum(not s for s, _ in verdicts)


def test_out_may_lie_beside_q_in_one_buffer(lib):
    """Rows of 2 heads of 16 in a buffer of 64 columns: q in the first 32, out in the others.  (What is not refused for
    its place is refused for a missing workspace.)"""
    big = dict(max_pages=4096, page_size=64, num_pages=1, keys=BASE + (1 << 24), values=BASE + (1 << 26), workspace=None, q=BASE,
               q_token_stride=64, out_token_stride=64)
    assert lib.dc_paged_attention(attention_args(BASE, out=BASE + 2 * 32, **big), 1, None) == -4
    for column in (0, 8, 16, 24, 40, 48, 56):  # the last ones reach into the next token's q
        assert lib.dc_paged_attention(attention_args(BASE, out=BASE + 2 * column, **big), 1, None) == -3, column
        assert b"overlaps an operand" in lib.dc_last_error()
