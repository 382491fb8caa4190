"""Frame attention where its operators and its layer can go wrong beside the ordinary cases: long caches with one
dominant slot, scores far from zero, graphs and eager frames of one layer."""
import math

import pytest
import torch

import frame_reference as ref
from test_gpu_frame_attention import DTYPES, PlainFrames, _layer, ids, make_pool, poison_unused, starts_of, widened
from util import DEV

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("streams,tokens", [(32, 1), (64, 70)], ids=["rows of 32", "rows of 128"])
def test_paged_attention_many_small_probabilities_beside_a_large_one(lib, streams, tokens):
    """One slot scores 17.375 above 130559 equal ones (each 2^-25.07 of it) whose values are 1, its own are 0; so many
    workgroups that none shares its slots.  out = n e / (1 + n e), e = exp(-17.375).

    A probability in fp16 is off by 2^-11 of itself or by 2^-32 of the largest, whichever is more: n 2^-32 in all.
    Their sum is exact: equal multiples of 2^-24 below 2^7, at most 2^6 units each and 2^23 together.  The
    normaliser adds up n / 32 blocks and 4 pieces: 2 (n / 32 + 16) w; exponentials and quotient 16 w; the result 2^-11."""
    from deltacnn_amd import hip_kernels as hk
    n, kv, dim, page, gap = 130560, 8, 64, 64, 17.375
    keys = torch.zeros(n // page, kv, page, dim, dtype=torch.float16, device=DEV)
    values = torch.ones_like(keys)
    keys[0, :, 3, 0] = gap
    values[0, :, 3] = 0
    table = torch.arange(n // page, dtype=torch.int32, device=DEV).expand(streams, n // page).contiguous()  # read by all
    q = torch.zeros(streams * tokens, kv, dim, dtype=torch.float16, device=DEV)
    q[..., 0] = 1
    lens = torch.full((streams,), n, dtype=torch.int32, device=DEV)
    got, lse = hk.paged_attention(q, keys, values, table, lens, scale=1.0, return_lse=True)
    assert b"join" not in lib.dc_last_kernels()
    mass = (n - 1) * math.exp(-gap)
    want = mass / (1 + mass)
    u = ref.half_step(torch.float16)
    tol = n * 2.0 ** -32 + want * (2 * u + (2 * (n / 32 + 16) + 16) * ref.W)
    assert float((got.double() - want).abs().max()) <= tol
    assert float((lse.double() - gap - math.log1p(mass)).abs().max()) <= (n / 32 + 16 + 8 * (gap + 2)) * ref.W


@pytest.mark.parametrize("tokens,wide", [(1, False), (150, False), (150, True)])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_paged_attention_equal_scores_far_from_zero(lib, tokens, wide, sign):
    """Scores of one value up to 2^32, where a step of fp32 is 2^8 and more: every slot counts the same, and nothing
    overflows fp16.  All probabilities are one number, rounded once: (u + 2 n w + 16 w) mean |v| + u |out|.

    That holds where the number is a normal one in fp16.  The maximum that is subtracted, in powers of two, is
    off by half a step at most, 2^3 below 2^28: the number is 2^-8 or more.  From 2^28 on half a step is 2^4 and more, a
    score is good to no power of two, and any weights of the slots are as good: what is left is |out| <= max |v|."""
    from deltacnn_amd import hip_kernels as hk
    gen = torch.Generator().manual_seed(50)
    n, dim, page = 300, 64, 32
    keys, values, _, _, table = make_pool(gen, 1, n, 1, page, dim, torch.float16)
    table = widened(table, page, tokens, 1, 1) if wide else table
    v = ref.gather(values, table[0], n, 0, page)
    want, u = v.mean(0), ref.half_step(torch.float16)
    tol = (u + (2 * n + 16) * ref.W) * v.abs().mean(0) + u * want.abs()
    q = torch.zeros(tokens, 1, dim, dtype=torch.float16)
    lens = torch.tensor([n], dtype=torch.int32, device=DEV)
    keys.zero_()
    for power in range(10, 32):
        q[..., 0] = min(1.37 * 2.0 ** (power // 2), 61000.0)
        keys[..., 0] = sign * min(1.23 * 2.0 ** (power - power // 2), 63000.0)
        got = hk.paged_attention(q.to(DEV), keys.to(DEV), values.to(DEV), table.to(DEV), lens, scale=1.0)
        if float(q[0, 0, 0]) * abs(float(keys[0, 0, 0, 0])) * math.log2(math.e) < 2.0 ** 28:
            ref.assert_within(got[:, 0], want.expand(tokens, dim), tol.expand(tokens, dim), f"2^{power}")
        else:
            assert float(got.abs().nan_to_num(math.inf).max()) <= float(v.abs().max()), f"2^{power}"


# ---- streams without tokens ----

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bfloat16", "float32"])
@pytest.mark.parametrize("active", [1, 20])
def test_paged_attention_where_most_streams_wait(lib, dtype, active):
    """Fewer rows than streams: the slot axis is still cut into pieces."""
    from deltacnn_amd import hip_kernels as hk
    gen = torch.Generator().manual_seed(80 + active)
    streams, n, dim, page = 32, 2000, 64, 64
    chosen = sorted(torch.randperm(streams, generator=gen)[:active].tolist())
    counts = [int(b in chosen) for b in range(streams)]
    lens = [n - 7 * b if counts[b] else 5 for b in range(streams)]
    keys, values, weights, _, table = make_pool(gen, streams, n, 1, page, dim, dtype)
    q = (1.5 * torch.randn(active, 1, dim, generator=gen)).to(dtype)
    lens_t, starts = torch.tensor(lens, dtype=torch.int32), starts_of(counts)
    out, tol, lse, lse_tol, ww, w_tol = ref.attention(q, keys, values, table, lens_t, starts, None, 0, weights, 0.75)
    w = weights.to(DEV)
    got, got_lse = hk.paged_attention(*(t.to(DEV) for t in (q, keys, values, table, lens_t)), starts=starts.to(DEV), weights=w,
                                      decay=0.75, return_lse=True)
    assert b"attention_join_kernel" in lib.dc_last_kernels()
    ref.assert_within(got, out, tol, "out")
    ref.assert_within(got_lse, lse, lse_tol, "lse")
    ref.assert_within(w, ww, w_tol, "weights")


# ---- rows of more than 256 bytes, 33 .. 64 a stream and head: two wavefronts a workgroup ----

NARROW = [  # counts, lens, q_heads, kv_heads, page, causal_block
    ([40], [300], 1, 1, 64, 0), ([64], [333], 1, 1, 33, 1), ([33], [200], 1, 1, 13, 0), ([25, 20], [190, 90], 2, 1, 16, 5),
    ([50, 0, 20, 64], [77, 9, 150, 64], 2, 2, 64, 16), ([50, 3, 64], [40, 3, 300], 1, 1, 13, 1), ([64], [1], 3, 3, 1, 0),
    ([45], [31], 1, 1, 33, 7),
]


@pytest.mark.parametrize("dtype,dim", [(torch.float16, 256), (torch.bfloat16, 256), (torch.bfloat16, 136), (torch.float32, 256),
                                       (torch.float32, 136), (torch.float32, 96)], ids=str)
@pytest.mark.parametrize("shape", NARROW, ids=str)
def test_paged_attention_two_wavefronts(lib, dtype, dim, shape):
    from deltacnn_amd import hip_kernels as hk
    counts, lens, heads, kv, page, block = shape
    gen = torch.Generator().manual_seed(3000 + sum(counts) + sum(lens))
    streams = len(counts)
    assert 32 * streams < sum(counts) * (heads // kv) <= 64 * streams
    keys, values, weights, _, table = make_pool(gen, streams, max(lens) + page, kv, page, dim, dtype)
    poison_unused(keys, values, weights, table, lens, page)
    q = (1.5 * torch.randn(sum(counts), heads, dim, generator=gen)).to(dtype)
    for b, n in enumerate(lens):
        table[b, -(-n // page):] = -12345
    lens_t, starts = torch.tensor(lens, dtype=torch.int32), starts_of(counts)
    out, tol, lse, lse_tol, ww, w_tol = ref.attention(q, keys, values, table, lens_t, starts, None, block, weights, 0.75)
    w = weights.to(DEV)
    got, got_lse = hk.paged_attention(*(t.to(DEV) for t in (q, keys, values, table, lens_t)),
                                      starts=starts.to(DEV) if len(set(counts)) > 1 else None, causal_block=block, weights=w, decay=0.75, return_lse=True)
    ref.assert_within(got, out, tol, "out")
    ref.assert_within(got_lse, lse, lse_tol, "lse")
    ref.assert_within(w, ww, w_tol, "weights")


@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("block", [0, 1])
def test_paged_attention_two_wavefronts_over_long_pieces(lib, dtype, block):
    """Four streams of 8 heads share the card: pieces of more blocks than the rings of tiles hold."""
    from deltacnn_amd import hip_kernels as hk
    gen = torch.Generator().manual_seed(90)
    tokens, kv, dim, page, lens = 40, 8, 256, 64, [6400, 3333, 1, 5001]
    keys, values, _, _, table = make_pool(gen, 4, max(lens), kv, page, dim, dtype)
    q = (1.5 * torch.randn(4 * tokens, kv, dim, generator=gen)).to(dtype)
    lens_t = torch.tensor(lens, dtype=torch.int32)
    out, tol, lse, lse_tol, _, _ = ref.attention(q, keys, values, table, lens_t, None, None, block)
    got, got_lse = hk.paged_attention(*(t.to(DEV) for t in (q, keys, values, table, lens_t)), causal_block=block, return_lse=True)
    ref.assert_within(got, out, tol, "out")
    ref.assert_within(got_lse, lse, lse_tol, "lse")


# ---- one buffer for all ----

@pytest.mark.parametrize("tokens", [1, 2, 21])
@pytest.mark.parametrize("order", ["t x h d", "t h x d", "h t x d", "h x t d", "x t h d", "x h t d"])
def test_rotary_append_in_place_of_any_projection(lib, tokens, order):
    """q, k and v in one buffer, dimensions in any order, q turned in place: as with tensors of their own."""
    from deltacnn_amd import hip_kernels as hk
    gen = torch.Generator().manual_seed(70)
    heads, dim, page = 3, 16, 8
    own = torch.randn(3, tokens, heads, dim, generator=gen).half().to(DEV)
    names = order.split()
    at = [("x", "t", "h", "d").index(n) for n in names]
    fused = own.permute(at).contiguous()
    q, k, v = fused.permute([names.index(n) for n in ("x", "t", "h", "d")])
    pos = torch.randint(-40, 40, (tokens, 2), generator=gen, dtype=torch.int32).to(DEV)
    freq = hk.rotary_frequencies((8, 8), device=DEV)
    table = torch.arange(4, dtype=torch.int32, device=DEV)[None]
    slots = torch.arange(tokens, dtype=torch.int32, device=DEV).expand(heads, tokens).contiguous()
    pools = [[torch.zeros(4, heads, page, dim, dtype=torch.float16, device=DEV) for _ in range(2)] for _ in range(2)]
    want = hk.rotary_append(*own, pos, freq, (8, 8), *pools[0], table, slots)
    got = hk.rotary_append(q, k, v, pos, freq, (8, 8), *pools[1], table, slots, out=q)
    assert got.data_ptr() == q.data_ptr() and torch.equal(got, want)
    assert torch.equal(k, own[1]) and torch.equal(v, own[2])
    assert all(torch.equal(a, b) for a, b in zip(*pools))


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["float16", "float32"])
@pytest.mark.parametrize("tokens", [1, 90])
def test_paged_attention_beside_its_queries(lib, dtype, tokens):
    """q and out as columns of one buffer: as with a tensor of its own, and q stays."""
    from deltacnn_amd import hip_kernels as hk
    gen = torch.Generator().manual_seed(71)
    heads, dim, n = 4, 64, 500
    keys, values, weights, _, table = (t.to(DEV) for t in make_pool(gen, 1, n, 2, 64, dim, dtype))
    both = torch.randn(tokens, 2 * heads, dim, generator=gen).to(dtype).to(DEV)
    q, out = both.split(heads, 1)
    own = q.clone()
    lens = torch.tensor([n], dtype=torch.int32, device=DEV)
    w = weights.clone()
    want = hk.paged_attention(own, keys, values, table, lens, weights=w)
    got = hk.paged_attention(q, keys, values, table, lens, weights=weights, out=out)
    assert got.data_ptr() == out.data_ptr() and torch.equal(got, want) and torch.equal(q, own) and torch.equal(weights, w)


# ---- the layer ----

def frames_of(shape, count, seed, dtype=torch.float16):
    gen = torch.Generator().manual_seed(seed)
    return [torch.randn(shape, generator=gen).to(dtype).to(DEV).contiguous(memory_format=torch.channels_last) for _ in range(count)]


def test_a_graph_keeps_its_state_beside_eager_frames_of_another_size(lib):
    """A frame of another size starts a new state; the graph goes on with its own, and what is allocated in
    between is not written to."""
    from deltacnn_amd.graph import FrameGraph
    video, other = frames_of((2, 48, 3, 3), 7, 60), frames_of((1, 48, 5, 4), 7, 61)
    layer, eager, eager_other = (_layer(torch.float16) for _ in range(3))
    with torch.no_grad():
        wanted, wanted_other = [eager(x).clone() for x in video], [eager_other(x).clone() for x in other]
        assert torch.equal(layer(video[0]), wanted[0])
        graph = FrameGraph(layer, video[0])
        kept = []
        for t in range(1, 7):
            assert torch.equal(layer(other[t - 1]), wanted_other[t - 1])
            kept += [torch.full((n,), 77, dtype=torch.int32, device=DEV) for n in (1, 2, 4, 8, 54, 128, 1024, 4096)]
            got = graph(video[t]).clone()
            torch.cuda.synchronize()
            assert torch.equal(got, wanted[t]), f"frame {t}"
            assert all(bool((k == 77).all()) for k in kept)


def test_the_first_frame_of_a_size_is_not_captured(lib):
    """The state has to be there before the capture; a refused capture leaves layer and stream usable."""
    from deltacnn_amd.graph import FrameGraph
    video, other = frames_of((2, 48, 3, 3), 3, 62), frames_of((1, 48, 5, 4), 1, 63)
    layer, eager = _layer(torch.float16), _layer(torch.float16)
    with torch.no_grad():
        with pytest.raises(RuntimeError, match="before the capture"):
            FrameGraph(layer, video[0])
        wanted = [eager(x).clone() for x in video]
        assert torch.equal(layer(video[0]), wanted[0])
        with pytest.raises(RuntimeError, match="before the capture"):
            FrameGraph(layer, other[0])
        assert torch.equal(layer(video[1]), wanted[1])  # the refused frame has changed nothing
        graph = FrameGraph(layer, video[0])
        assert torch.equal(graph(video[2]), wanted[2])


class Protecting:
    """A layer as PlainFrames wants to see it, which counts the frame that arrives among `keep_frames`: one more."""

    def __init__(self, layer):
        self.layer, self.keep_frames = layer, layer.keep_frames + 1

    def __getattr__(self, name):
        return getattr(self.layer, name)


@pytest.mark.parametrize("keep", [0, 1, 2])
def test_layer_protects_the_last_frames(lib, keep):
    """fp32, two streams, eight frames of which four fit: the tokens of the last `keep` frames stay whatever attention
    they have received, in every kv head, and outputs, slots and stamps are those of the 64-bit statement.

    Its numbers are sums of at most 48 (projections) and 80 (slots) terms of magnitude about 1 in fp32 behind two
    projections: 10 (48 + 80) w relative to outputs below 1; weights that decide have to differ by twice that."""
    from deltacnn_amd.sparse_layers import DCFrameAttention
    torch.manual_seed(4)
    layer = DCFrameAttention(48, 4, kv_heads=2, head_dim=24, frames=4, keep_frames=keep, decay=0.5, page_size=16).eval().to(DEV)
    shape = (2, 48, 4, 5)
    plain = PlainFrames(Protecting(layer), shape)
    gen = torch.Generator().manual_seed(8)
    rescued = 0
    with torch.no_grad():
        for t in range(8):
            x = torch.randn(shape, generator=gen)
            before = [[[(c, c[2]) for c in cells] for cells in heads] for heads in plain.kept]
            want = plain.frame(x)
            got = layer(x.to(DEV).contiguous(memory_format=torch.channels_last))
            assert float((got.double().cpu() - want).abs().max()) < 10 * 128 * ref.W, f"frame {t}"
            s = layer._state
            for b in range(2):
                for h in range(2):
                    cells = plain.kept[b][h]
                    stamps = ref.gather(s["stamps"].cpu()[..., None], s["table"].cpu()[b], len(cells), h, 16)[:, 0]
                    assert stamps.tolist() == [c[3] for c in cells], f"frame {t}: other tokens were kept"
                    for back in range(min(keep, t) + 1):
                        assert int((stamps == t - back).sum()) == 20, f"frame {t}: tokens of frame {t - back} went"
                    gone = [w for c, w in before[b][h] if not any(c is d for d in cells)]
                    if gone:
                        rescued += sum(w < max(gone) for c, w in before[b][h] if t - keep <= c[3])
    assert 20 * 128 * ref.W < plain.gap < math.inf
    assert (rescued > 0) == (keep > 0)  # without the protection other tokens would have gone


def test_layer_lets_go_of_an_earlier_scene(lib):
    """With the constructor's own decay and protection, 40 frames of one scene are gone after as many frames of
    another as the cache holds.

    Queries and keys are 4 x and 4 x (but for the one pair that turns with the position), x is +1 or -1: a score is +-34,
    so that a frame attends to its own scene alone, evenly.  With decay d a token of the first scene has at most
    1 (its first frame) + 1 / (F (1 - d)), F = 4 frames in the cache; d = 0.5 makes that 1.5 and halves it with every
    frame of the second scene, whose j-th frame gives each of its j n tokens 1 / j.  When frame j = 3, 4 chooses, the first
    scene's tokens are below 1.5 / 2^(j - 1) < 1 / 2, the second's in front of the protected frame above 1 / 2 + 1 / 2."""
    from deltacnn_amd.sparse_layers import DCFrameAttention
    layer = DCFrameAttention(8, 1, frames=4, sections=(2, 0, 0), page_size=16).eval()
    with torch.no_grad():
        layer.qkv.weight.zero_()
        layer.qkv.bias.zero_()
        for e in range(2, 8):
            layer.qkv.weight[e, e] = layer.qkv.weight[8 + e, e] = 4.0
        layer.qkv.weight[16:24] = torch.eye(8)
        layer.to(DEV)
        x = torch.ones(1, 8, 3, 3, device=DEV).contiguous(memory_format=torch.channels_last)
        for _ in range(40):
            layer(x)
        for _ in range(4):
            layer(-x)
    s = layer._state
    stamps = ref.gather(s["stamps"].cpu()[..., None], s["table"].cpu()[0], 36, 0, 16)[:, 0]
    assert sorted(stamps.tolist()) == [t for t in range(40, 44) for _ in range(9)]


def test_alternating_sizes_do_not_grow_memory(lib):
    from deltacnn_amd.sparse_layers import DCModule
    layer = _layer(torch.float16)
    one, two = frames_of((1, 48, 3, 3), 1, 64)[0], frames_of((2, 48, 3, 3), 1, 65)[0]
    before, seen = DCModule.get_temp_buffer_numel(), []
    with torch.no_grad():
        for _ in range(4):
            layer(one)
            layer(two)
            torch.cuda.synchronize()
            seen.append((DCModule.get_temp_buffer_numel() - before, torch.cuda.memory_allocated()))
    assert seen[0][0] > 0 and all(x == seen[0] for x in seen)


def test_frames_in_inference_mode_and_out_of_it(lib):
    video = frames_of((1, 48, 3, 3), 6, 66)
    layer, eager = _layer(torch.float16), _layer(torch.float16)
    with torch.no_grad():
        wanted = [eager(x).clone() for x in video]
    for t, x in enumerate(video):
        with torch.inference_mode() if t % 2 == 0 else torch.no_grad():
            assert torch.equal(layer(x), wanted[t]), f"frame {t}"
