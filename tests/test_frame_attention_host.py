"""Frame attention without a GPU: what the entry points refuse, before anything is launched, and the
arithmetic that the kernels' shortcuts rest on."""
import ctypes
import math

import numpy as np
import pytest
import torch

import frame_reference as ref


def _buf():
    raw = (ctypes.c_char * 8192)()
    return raw, (ctypes.addressof(raw) + 15) // 16 * 16


def rotary_args(p, **kw):
    from deltacnn_amd._lib import RotaryArgs
    a = RotaryArgs(4, 2, 1, 16, p, 32, 16, p + 4096, 32, 16, p, 2, (ctypes.c_int32 * 4)(8, 8, 0, 0), p, 0, 0, p, p, 16, 16, 16, 16, p, p,
                   p, p, None, p, p, None, 2, 3, 8, 2, p, p)
    for k, v in kw.items():
        if k == "sections":
            a.sections[:] = v
        else:
            setattr(a, k, v)
    return ctypes.byref(a)


def attention_args(p, **kw):
    from deltacnn_amd._lib import AttentionArgs
    a = AttentionArgs(4, 2, 1, 16, p, 32, 16, p + 4096, 32, 16, None, p, p, p, p, None, 2, 1, 8, 2, 0, 0.25, None, 1.0, p, 1 << 30)
    for k, v in kw.items():
        setattr(a, k, v)
    return ctypes.byref(a)


def slots_args(p, **kw):
    from deltacnn_amd._lib import SlotsArgs
    a = SlotsArgs(p, p, p, p, p, None, 2, 4, 1, 3, 8, 2, 10, p, p + 64, p, 1 << 30)
    for k, v in kw.items():
        setattr(a, k, v)
    return ctypes.byref(a)


@pytest.mark.parametrize("change,code", [
    (dict(tokens=0), -2), (dict(q_heads=0), -2), (dict(dim=-1), -2), (dict(q_heads=2000), -3), (dict(tokens=1 << 25), -3),
    (dict(dim=2048), -3), (dict(axes=0), -2), (dict(axes=5), -2), (dict(sections=(7, 8, 0, 0)), -2), (dict(sections=(-2, 8, 0, 0)), -2),
    (dict(sections=(12, 8, 0, 0)), -2), (dict(sections=(0, 0, 0, 0)), -2), (dict(q=None), -4), (dict(out=None), -4), (dict(positions=None), -4),
    (dict(frequencies=None), -4), (dict(q_token_stride=8), -2), (dict(q_head_stride=8), -2), (dict(values=None), -4), (dict(slots=None), -4),
    (dict(page_table=None), -4), (dict(k=None), -4), (dict(k_token_stride=3), -2), (dict(new_lens=None), -4), (dict(page_size=0), -2),
    (dict(num_pages=0), -2), (dict(streams=3), -2), (dict(streams=70000, tokens=70000), -3), (dict(max_pages=1 << 28), -3),
], ids=str)
def test_rotary_refuses(lib, change, code):
    raw, p = _buf()
    assert lib.dc_rotary(rotary_args(p, **change), 1, None) == code, lib.dc_last_error()
    assert lib.dc_last_kernels() == b""


def test_rotary_refuses_types_alignment_and_overlap(lib):
    raw, p = _buf()
    assert lib.dc_rotary(None, 1, None) == -4
    assert lib.dc_rotary(rotary_args(p), 9, None) == -1
    assert lib.dc_rotary(rotary_args(p, q=p + 1), 1, None) == -5
    assert lib.dc_rotary(rotary_args(p, frequencies=p + 4), 1, None) == -5
    assert lib.dc_rotary(rotary_args(p, slots=p + 2), 1, None) == -5
    # out: q itself is fine (nothing is refused before the launch), other overlaps are not
    for change in (dict(out=p + 2), dict(out=p, out_token_stride=48), dict(out=p + 32 * 2 + 8)):
        assert lib.dc_rotary(rotary_args(p, keys=None, **change), 1, None) == -3, change
    # columns of one wider buffer interleave without touching: refused only where they touch
    wide = dict(keys=None, q_token_stride=64, out_token_stride=64)
    assert lib.dc_rotary(rotary_args(p, out=p + 48 * 2, **wide), 1, None) == -3
    assert lib.dc_rotary(rotary_args(p, out=p + 16 * 2, **wide), 1, None) == -3
    # the cache's write: out over k or v, anything over the cache, keys over values, rows of out over each other
    apart = dict(k=p + 1024, v=p + 1024, keys=p + 4352, values=p + 6144, weights=p + 2048, stamps=p + 2048)  # a pool has 3 x 8 x 16 elements
    for change, what in ((dict(out=p + 1024), b"out overlaps k"), (dict(out=p + 512, k=p + 256, v=p + 640), b"out overlaps k or v"),
                         (dict(k=p + 4400), b"overlaps the cache"), (dict(keys=p + 64), b"overlaps the cache"), (dict(weights=p + 6144), b"overlaps the cache"),
                         (dict(values=p + 4352), b"keys and values overlap")):
        assert lib.dc_rotary(rotary_args(p, **{**apart, **change}), 1, None) == -3 and what in lib.dc_last_error(), change
    assert lib.dc_rotary(rotary_args(p, keys=None, out_token_stride=16), 1, None) == -3
    assert lib.dc_rotary(rotary_args(p, tokens=1 << 21, q_heads=1024), 1, None) == -3
    assert lib.dc_last_kernels() == b""


@pytest.mark.parametrize("change,code", [
    (dict(tokens=0), -2), (dict(kv_heads=0), -2), (dict(q_heads=3, kv_heads=2), -2), (dict(dim=12), -3), (dict(dim=264), -3), (dict(dim=0), -2),
    (dict(streams=3), -2), (dict(page_size=0), -2), (dict(max_pages=0), -2), (dict(num_pages=-1), -2), (dict(causal_block=-1), -2),
    (dict(scale=math.nan), -3), (dict(decay=math.nan), -3), (dict(q=None), -4), (dict(out=None), -4), (dict(keys=None), -4), (dict(values=None), -4),
    (dict(lens=None), -4), (dict(page_table=None), -4), (dict(q_token_stride=8), -2), (dict(q_token_stride=33), -5), (dict(q_head_stride=17), -5),
    (dict(max_pages=1 << 28), -3), (dict(weights=1, workspace=None), -5), (dict(kv_heads=300, q_heads=300), -3),
], ids=str)
def test_paged_attention_refuses(lib, change, code):
    raw, p = _buf()
    assert lib.dc_paged_attention(attention_args(p, **change), 1, None) == code, lib.dc_last_error()
    assert lib.dc_last_kernels() == b""


def test_paged_attention_refuses_types_alignment_and_overlap(lib):
    raw, p = _buf()
    assert lib.dc_paged_attention(None, 1, None) == -4
    assert lib.dc_paged_attention(attention_args(p), 3, None) == -1
    assert lib.dc_paged_attention_workspace(attention_args(p), 3) == -1
    assert lib.dc_paged_attention(attention_args(p, q=p + 8), 1, None) == -5
    assert lib.dc_paged_attention(attention_args(p, keys=p + 8), 1, None) == -5
    assert lib.dc_paged_attention(attention_args(p, out=p + 4097), 1, None) == -5
    assert lib.dc_paged_attention(attention_args(p, out=p), 1, None) == -3
    assert lib.dc_paged_attention(attention_args(p, out=p + 64, keys=p + 2048, values=p + 2048), 1, None) == -3  # over q
    assert lib.dc_paged_attention(attention_args(p, out_token_stride=16), 1, None) == -3  # rows of out over each other
    assert lib.dc_paged_attention(attention_args(p, tokens=1 << 21, q_heads=1024), 1, None) == -3
    # a call that needs a workspace and has none, or too little
    big = dict(max_pages=4096, page_size=64, num_pages=1)
    need = lib.dc_paged_attention_workspace(attention_args(p, **big), 1)
    assert need > 0
    assert lib.dc_paged_attention(attention_args(p, workspace=None, **big), 1, None) == -4
    assert lib.dc_paged_attention(attention_args(p, workspace_bytes=need - 1, **big), 1, None) == -4
    assert lib.dc_paged_attention(attention_args(p, workspace=p + 4, **big), 1, None) == -5


@pytest.mark.parametrize("change,code", [
    (dict(tokens=0), -2), (dict(kv_heads=0), -2), (dict(streams=3), -2), (dict(budget=0), -2), (dict(budget=17), -2), (dict(page_size=-1), -2),
    (dict(weights=None), -4), (dict(lens=None), -4), (dict(slots=None), -4), (dict(new_lens=None), -4), (dict(keep_from=None), -4),
    (dict(page_table=None), -4), (dict(max_pages=1 << 28), -3),
], ids=str)
def test_cache_slots_refuses(lib, change, code):
    raw, p = _buf()
    assert lib.dc_cache_slots(slots_args(p, **change), None) == code, lib.dc_last_error()
    assert lib.dc_last_kernels() == b""


def test_cache_slots_refuses_alignment_overlap_and_a_missing_workspace(lib):
    raw, p = _buf()
    assert lib.dc_cache_slots(None, None) == -4
    assert lib.dc_cache_slots(slots_args(p, weights=p + 2), None) == -5
    assert lib.dc_cache_slots(slots_args(p, new_lens=p + 4), None) == -3
    big = dict(max_pages=1024, page_size=64)
    need = lib.dc_cache_slots_workspace(slots_args(p, **big))
    assert need > 0 and lib.dc_cache_slots_workspace(slots_args(p)) == 0
    assert lib.dc_cache_slots(slots_args(p, workspace=None, **big), None) == -4
    assert lib.dc_cache_slots(slots_args(p, workspace_bytes=need - 1, **big), None) == -4


def test_the_python_entry_points_refuse_host_tensors(lib):
    from deltacnn_amd import _lib
    from deltacnn_amd import hip_kernels as hk
    x, pos, f = torch.zeros(3, 2, 16), torch.zeros(3, 1, dtype=torch.int32), torch.zeros(8, dtype=torch.float64)
    pool, table, lens = torch.zeros(2, 2, 4, 16), torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    for call in (lambda: hk.rotary(x, pos, f, (16,)),
                 lambda: hk.rotary_append(x, x, x, pos, f, (16,), pool, pool, table, torch.zeros(2, 3, dtype=torch.int32)),
                 lambda: hk.paged_attention(x, pool, pool, table, lens),
                 lambda: hk.cache_slots(pool[..., 0], table, lens, 3, 8)):
        with pytest.raises(_lib.DeltaCNNError, match="GPU"):
            call()
    for bad in (None, 3, torch.zeros(4), torch.zeros(0, 2, 16)):
        with pytest.raises(_lib.DeltaCNNError):
            hk.rotary(bad, pos, f, (16,))
    with pytest.raises(_lib.DeltaCNNError, match="even"):
        hk.rotary_frequencies((3, 4))
    assert hk.rotary_frequencies((4, 0, 2), base=100.0).tolist() == [1.0, 0.1, 1.0]
    for bad in (1 << 31, -(1 << 31) - 1, 1 << 32):  # a field of the C interface would hold something else
        with pytest.raises(_lib.DeltaCNNError, match="32 bits"):
            hk._fits("paged_attention", 3, bad, 5)
    hk._fits("paged_attention", (1 << 31) - 1, -(1 << 31))
    with pytest.raises(ValueError):
        from deltacnn_amd.sparse_layers import DCFrameAttention
        DCFrameAttention(64, 4, kv_heads=3)


# ---- the arithmetic of the shortcuts ----

def test_division_by_multiplication_is_exact():
    """quotient = (n m) >> (31 + l), l = ceil(log2 d), m = ceil(2^(31 + l) / d), for 0 <= n < 2^31."""
    rng = np.random.default_rng(1)
    divisors = list(range(1, 300)) + [2 ** k + e for k in range(8, 31) for e in (-1, 0, 1)] + rng.integers(1, 2 ** 31, 300).tolist()
    for d in divisors:
        if not 1 <= d < 2 ** 31:
            continue
        l = (d - 1).bit_length()
        m = -(-(1 << (31 + l)) // d)
        assert m < 1 << 32
        top = (2 ** 31 - 1) // d
        for q in {0, 1, top // 2, top - 1, top, *rng.integers(0, top + 1, 5).tolist()}:
            for n in (q * d - 1, q * d, q * d + 1):
                if 0 <= n < 2 ** 31:
                    assert n * m >> (31 + l) == n // d, (n, d)


@pytest.mark.parametrize("exponent", [0x7c00, 0x7f80], ids=hex)
def test_odd_elements_of_a_word(exponent):
    """Two 16-bit elements at once: infinities and NaN, and nothing else, lose their bits."""
    low = np.arange(1 << 16, dtype=np.uint64)
    both = exponent << 16 | exponent
    for high in [0, 1, 0x8000, 0xffff, 0x7fff, exponent, exponent | 1, exponent ^ 0x8000, exponent - 1, exponent + 1, exponent & ~0x100, 0x3c00, 0x3f80]:
        for w in (low | np.uint64(high) << np.uint64(16), low << np.uint64(16) | np.uint64(high)):
            x = (w & both) ^ both
            bits = (x - 0x00010001) % (1 << 32) & ~x & 0x80008000
            kept = w & ~((bits >> np.uint64(15)) * np.uint64(0xffff))
            for shift in (0, 16):
                e = w >> np.uint64(shift) & np.uint64(0xffff)
                odd = (e & exponent) == exponent
                assert np.array_equal(kept >> np.uint64(shift) & np.uint64(0xffff), np.where(odd, 0, e))


def test_tile_places_hit_every_bank_once():
    """Keys: 16 rows' chunks of one operand; values: 32 lanes of the transposing read.  256 bytes each, all different."""
    for row_bytes in (128, 256, 512, 1024):
        chunks = row_bytes // 16
        key = lambda r: r & 15 if row_bytes >= 256 else r >> 1 & 7  # noqa: E731
        for c in range(chunks):
            for r0 in (0, 16):
                assert len({(r * row_bytes + ((c ^ key(r)) << 4)) % 256 for r in range(r0, r0 + 16)}) == 16
        for r in range(64):
            assert sorted(c ^ key(r) for c in range(chunks)) == list(range(chunks))
    for row_bytes, dim in ((128, 64), (256, 128), (512, 256)):
        value = lambda r: (r & 3) << 2 if dim >= 128 else (r & 2) << 1  # noqa: E731
        for r0 in range(0, 32, 4):
            for c0 in range(0, row_bytes // 16, 4):
                assert len({(r * row_bytes + ((c ^ value(r)) << 4)) % 256 for r in range(r0, r0 + 4) for c in range(c0, c0 + 4)}) == 16


def test_operand_order_of_the_two_products():
    """What a lane holds of S^T (rows 8 (r / 4) + 4 half + r % 4) is what it needs of P^T for the slots that
    two transposing reads at 16 t + 8 e + 4 half deliver."""
    for half in (0, 1):
        for t in (0, 1):
            held = [8 * (r // 4) + 4 * half + r % 4 for r in range(8 * t, 8 * t + 8)]
            read = [16 * t + 8 * e + 4 * half + i for e in (0, 1) for i in range(4)]
            assert held == read


# ---- the oracle ----

def test_oracle_attention_against_torch():
    gen = torch.Generator().manual_seed(0)
    n, new, dim = 37, 6, 16
    keys, values = torch.randn(10, 1, 4, dim, generator=gen), torch.randn(10, 1, 4, dim, generator=gen)
    table = torch.arange(10, dtype=torch.int32).flip(0)[None].contiguous()
    q = torch.randn(new, 2, dim, generator=gen)
    lens = torch.tensor([n], dtype=torch.int32)
    k, v = ref.gather(keys, table[0], n, 0, 4), ref.gather(values, table[0], n, 0, 4)
    for block in (0, 1, 4):
        out, _, lse, _, w, _ = ref.attention(q, keys, values, table, lens, causal_block=block, weights=torch.zeros(10, 1, 4), decay=1.0)
        mask = torch.ones(new, n, dtype=torch.bool)
        if block:
            mask = torch.arange(n)[None] < (n - new + (torch.arange(new) // block + 1) * block)[:, None]
        want = torch.nn.functional.scaled_dot_product_attention(q.double().transpose(0, 1), k.expand(2, n, dim), v.expand(2, n, dim), attn_mask=mask)
        assert torch.allclose(out, want.transpose(0, 1), atol=1e-12)
        assert math.isclose(float(w.sum()), 2 * new, rel_tol=1e-12)


def test_oracle_rotation_keeps_lengths_and_its_gradient_is_the_inverse():
    gen = torch.Generator().manual_seed(3)
    x, y = torch.randn(4, 2, 12, generator=gen), torch.randn(4, 2, 12, generator=gen)
    pos = torch.randint(-50, 50, (4, 2), generator=gen, dtype=torch.int32)
    from deltacnn_amd import hip_kernels as hk
    f = hk.rotary_frequencies((4, 6))
    for interleaved in (False, True):
        turned = ref.rotary(x, pos, f, (4, 6), interleaved)[0]
        assert torch.allclose(turned.norm(dim=2), x.double().norm(dim=2))
        grad = ref.rotary(y, pos, f, (4, 6), interleaved, inverse=True)[0]  # of <turned, y>
        eps = 2.0 ** -10
        for i in range(12):  # differences: the rotation is linear, so they are exact up to rounding
            step = x.clone()
            step[:, :, i] += eps
            diff = ((ref.rotary(step, pos, f, (4, 6), interleaved)[0] - turned) * y.double()).sum(2) / (step - x).double()[:, :, i]
            assert torch.allclose(diff, grad[:, :, i], atol=1e-9)
