"""Rotary positions into a paged cache, attention over it and the choice of slots for new tokens,
against the 64-bit definition in frame_reference (bounds derived there)."""
import math

import pytest
import torch

import frame_reference as ref
from util import DEV

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16, torch.float32]
ids = lambda t: str(t)[6:] if isinstance(t, torch.dtype) else None  # noqa: E731


def make_pool(gen, streams, slots, kv, page, dim, dtype, spare=3):
    """Keys, values, weights, stamps and a page table whose pages are shuffled; what lies in no slot is NaN."""
    per = max(1, -(-slots // page))
    pages = streams * per + spare
    table = torch.randperm(pages, generator=gen)[:streams * per].view(streams, per).to(torch.int32)
    keys = torch.randn(pages, kv, page, dim, generator=gen).to(dtype)
    values = torch.randn(pages, kv, page, dim, generator=gen).to(dtype)
    weights = torch.rand(pages, kv, page, generator=gen)
    stamps = torch.randint(0, 9, (pages, kv, page), generator=gen, dtype=torch.int32)
    return keys, values, weights, stamps, table


def widened(table, page, tokens, heads, kv):
    """The same pages in a table with room for so many slots that a workgroup takes 128 rows, where a stream has more than 64."""
    streams = table.shape[0]
    blocks = -(-tokens * (heads // kv) // (32 * streams)) * streams * kv
    wide = torch.full((streams, max(table.shape[1], -(-29 * 1024 * 32 // (blocks * page)))), -12345, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    return wide


def poison_unused(keys, values, weights, table, lens, page):
    """NaN wherever no stream has a slot in use."""
    used = torch.zeros(keys.shape[0], page, dtype=torch.bool)
    for b, n in enumerate(lens):
        for s in range(n):
            used[int(table[b, s // page]), s % page] = True
    hole = ~used[:, None, :]
    keys.masked_fill_(hole[..., None], math.nan)
    values.masked_fill_(hole[..., None], math.nan)
    weights.masked_fill_(hole, math.nan)


def starts_of(counts):
    s = [0]
    for c in counts:
        s.append(s[-1] + c)
    return torch.tensor(s, dtype=torch.int32)


# ---- rotary ----

ROTARY = [  # tokens, heads, dim, sections
    (1, 1, 8, (8,)), (3, 2, 64, (16, 24, 24)), (33, 5, 128, (32, 48, 48)), (7, 3, 40, (10, 6)), (5, 1, 30, (2, 4, 6, 8)),
    (257, 4, 96, (0, 48, 48)), (19, 2, 72, (72,)), (2, 7, 256, (64, 64)), (65, 1, 17, (6,)),
]


@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shape", ROTARY, ids=str)
def test_rotary(lib, dtype, interleaved, shape):
    from deltacnn_amd import hip_kernels as hk
    tokens, heads, dim, sections = shape
    gen = torch.Generator().manual_seed(41 + tokens)
    x = torch.randn(tokens, heads, dim, generator=gen).to(dtype)
    pos = torch.randint(-5000000, 5000000, (tokens, len(sections)), generator=gen, dtype=torch.int32)
    freq = hk.rotary_frequencies(sections, device=DEV)
    for inverse in (False, True):
        want, tol = ref.rotary(x, pos, freq, sections, interleaved, inverse)
        got = hk.rotary(x.to(DEV), pos.to(DEV), freq, sections, interleaved=interleaved, inverse=inverse)
        ref.assert_within(got, want, tol, f"inverse={inverse}")
    # a strided view (heads in the outer dimension), in place
    buf = torch.full((heads + 1, tokens, dim + 3), 7.0, dtype=dtype, device=DEV)
    view = buf[1:, :, :dim].transpose(0, 1)
    view.copy_(x)
    got = hk.rotary(view, pos.to(DEV), freq, sections, interleaved=interleaved, out=view)
    want, tol = ref.rotary(x, pos, freq, sections, interleaved)
    ref.assert_within(view, want, tol, "in place")
    assert got.data_ptr() == view.data_ptr() and bool((buf[0] == 7).all()) and bool((buf[:, :, dim:] == 7).all())


def test_rotary_back_and_forth_and_its_gradient(lib):
    """inverse undoes the rotation, and is its transpose: <R x, y> = <x, R^-1 y>."""
    from deltacnn_amd import hip_kernels as hk
    gen = torch.Generator().manual_seed(5)
    sections, tokens = (8, 12, 12), 50
    x, y = (torch.randn(tokens, 3, 32, generator=gen).to(DEV) for _ in range(2))
    pos = torch.randint(0, 2000, (tokens, 3), generator=gen, dtype=torch.int32).to(DEV)
    freq = hk.rotary_frequencies(sections, device=DEV)
    turned = hk.rotary(x, pos, freq, sections)
    back = hk.rotary(turned, pos, freq, sections, inverse=True)
    # two turns of the bound of frame_reference.rotary: 2 * (7 + 1) w (|a| + |b|), |a| + |b| < 12
    assert float((back - x).abs().max()) < 16 * ref.W * 12
    lhs = (turned.double() * y.double()).sum()
    rhs = (x.double() * hk.rotary(y, pos, freq, sections, inverse=True).double()).sum()
    bound = 16 * ref.W * 2 * float((x.abs() * y.abs()).sum() + x.abs().sum() * 6)
    assert abs(float(lhs - rhs)) < bound


# ---- rotary_append ----

APPEND = [  # counts of new tokens, q_heads, kv_heads, dim, page, sections
    ([1], 4, 2, 64, 16, (16, 24, 24)), ([5, 5], 3, 3, 32, 7, (32,)), ([3, 0, 9], 8, 1, 128, 64, (32, 48, 48)),
    ([40, 1, 2, 17], 5, 5, 40, 30, (10, 6)), ([300], 2, 1, 96, 49, (48, 48)), ([70, 70, 70], 6, 2, 72, 1, (2, 2, 2)),
]


@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("shape", APPEND, ids=str)
def test_rotary_append(lib, dtype, shape):
    from deltacnn_amd import hip_kernels as hk
    counts, heads, kv, dim, page, sections = shape
    gen = torch.Generator().manual_seed(77 + sum(counts))
    tokens, streams = sum(counts), len(counts)
    behind = 3 if len(set(counts)) > 1 else 0  # tokens behind the last stream's
    total = tokens + behind
    slots_of = max(counts) + 11
    keys, values, weights, stamps, table = make_pool(gen, streams, slots_of, kv, page, dim, dtype)
    fused = torch.randn(total, (heads + 2 * kv) * dim, generator=gen).to(dtype)
    q = fused[:, :heads * dim].view(total, heads, dim)
    k = fused[:, heads * dim:(heads + kv) * dim].view(total, kv, dim)
    v = fused[:, (heads + kv) * dim:].view(total, kv, dim)
    pos = torch.randint(0, 100000, (total, len(sections)), generator=gen, dtype=torch.int32)
    starts = starts_of(counts)
    slots = torch.full((kv, total), -1, dtype=torch.int32)
    for b, (first, count) in enumerate(ref.spans(starts, streams, tokens)):
        for h in range(kv):
            slots[h, first:first + count] = torch.randperm(slots_of, generator=gen)[:count].to(torch.int32)
    if behind:
        slots[:, tokens:] = 0
    slots[0, 0] = -1                                       # a token that is not stored in head 0
    if tokens > 2:
        slots[kv - 1, 1] = table.shape[1] * page + 5       # ... and one beyond the stream's pages
    lost = int(table[streams - 1, 0])
    if streams > 1:
        table[streams - 1, 0] = 10 ** 6                    # a page outside the pool
    freq = hk.rotary_frequencies(sections)
    new_lens = torch.arange(1, streams + 1, dtype=torch.int32)
    want_q, q_tol = ref.rotary(q, pos, freq, sections, False)
    want_k, k_tol = ref.rotary(k, pos, freq, sections, False)
    wk, wv, ww, ws = keys.double(), values.clone(), weights.clone(), stamps.clone()
    tol = torch.zeros_like(wk)
    for b, (first, count) in enumerate(ref.spans(starts, streams, tokens)):
        for t in range(first, first + count):
            for h in range(kv):
                s = int(slots[h, t])
                if s < 0 or s >= table.shape[1] * page or not 0 <= int(table[b, s // page]) < keys.shape[0]:
                    continue
                pg, off = ref.place(table[b], s, page)
                wk[pg, h, off], tol[pg, h, off], wv[pg, h, off] = want_k[t, h], k_tol[t, h], v[t, h]
                ww[pg, h, off], ws[pg, h, off] = 0.0, pos[t, 0]
    d = {n: t.to(DEV) for n, t in dict(fused=fused, pos=pos, freq=freq, keys=keys, values=values, weights=weights, stamps=stamps,
                                       table=table, slots=slots, starts=starts, new=new_lens).items()}
    f = d["fused"]
    lens = torch.zeros(streams, dtype=torch.int32, device=DEV)
    got = hk.rotary_append(f[:, :heads * dim].view(total, heads, dim), f[:, heads * dim:(heads + kv) * dim].view(total, kv, dim),
                           f[:, (heads + kv) * dim:].view(total, kv, dim), d["pos"], d["freq"], sections, d["keys"], d["values"],
                           d["table"], d["slots"], starts=d["starts"] if len(set(counts)) > 1 else None, weights=d["weights"],
                           stamps=d["stamps"], lens=lens, new_lens=d["new"])
    ref.assert_within(got, want_q, q_tol, "q")
    ref.assert_within(d["keys"], wk, tol, "keys")
    assert torch.equal(d["values"].cpu(), wv) and torch.equal(d["weights"].cpu(), ww) and torch.equal(d["stamps"].cpu(), ws)
    assert lens.tolist() == new_lens.tolist()
    assert lost >= 0 and torch.equal(f.cpu(), fused)  # the inputs are left alone
    # stamps of the caller's own; no weights, no lens; q in place
    own = torch.arange(total, dtype=torch.int32, device=DEV) + 1000
    ws2 = ws.clone()
    for b, (first, count) in enumerate(ref.spans(starts, streams, tokens)):
        for t in range(first, first + count):
            for h in range(kv):
                s = int(slots[h, t])
                if 0 <= s < table.shape[1] * page and 0 <= int(table[b, s // page]) < keys.shape[0]:
                    pg, off = ref.place(table[b], s, page)
                    ws2[pg, h, off] = 1000 + t
    qv = f[:, :heads * dim].view(total, heads, dim)
    hk.rotary_append(qv, f[:, heads * dim:(heads + kv) * dim].view(total, kv, dim), f[:, (heads + kv) * dim:].view(total, kv, dim),
                     d["pos"], d["freq"], sections, d["keys"], d["values"], d["table"], d["slots"],
                     starts=d["starts"] if len(set(counts)) > 1 else None, stamps=d["stamps"], token_stamps=own, out=qv)
    ref.assert_within(qv, want_q, q_tol, "q in place")
    assert torch.equal(d["stamps"].cpu(), ws2)


@pytest.mark.parametrize("outer", ["tokens", "heads"])
def test_rotary_append_in_place_of_a_fused_projection(lib, outer):
    """q, k and v are columns of one buffer, token by token or head by head, and q is turned in place: the
    same as with tensors of their own, and k and v stay."""
    from deltacnn_amd import hip_kernels as hk
    gen = torch.Generator().manual_seed(41)
    tokens, heads, dim, page = 21, 3, 16, 8
    own = [torch.randn(tokens, heads, dim, generator=gen).half().to(DEV) for _ in range(3)]
    if outer == "tokens":
        fused = torch.cat(own, 1)
        q, k, v = fused.split(heads, 1)
    else:
        fused = torch.cat([t.transpose(0, 1) for t in own], 2).contiguous()
        q, k, v = (t.transpose(0, 1) for t in fused.split(dim, 2))
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


# ---- paged_attention ----

ATTEND = [  # counts, lens, q_heads, kv_heads, dim, page, causal_block
    ([1], [1], 1, 1, 8, 1, 0),
    ([1], [200], 5, 1, 64, 16, 0),
    ([1, 1, 1], [77, 0, 300], 8, 2, 128, 64, 0),
    ([1] * 9, [3, 64, 65, 63, 128, 1, 190, 5, 17], 4, 4, 40, 30, 0),
    ([4], [67], 2, 1, 32, 7, 0),
    ([49], [150], 4, 2, 64, 49, 0),
    ([49], [150], 4, 2, 64, 49, 7),
    ([33, 0, 70], [40, 20, 70], 3, 3, 96, 13, 1),
    ([130], [130], 2, 2, 64, 64, 1),
    ([130], [100], 2, 1, 64, 64, 1),           # more new tokens than slots: the first rows see nothing
    ([20], [9], 1, 1, 16, 4, 6),
    ([64, 64], [256, 256], 2, 2, 128, 64, 16),
    ([1], [1500], 16, 1, 256, 100, 0),
    ([90], [333], 1, 1, 256, 33, 30),
    ([2, 1, 3], [500, 31, 129], 20, 4, 72, 77, 0),
    ([300], [700], 2, 2, 128, 64, 0),
    ([17], [1100], 8, 8, 64, 196, 1),
]


@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("shape", ATTEND, ids=str)
def test_paged_attention(lib, dtype, shape):
    from deltacnn_amd import hip_kernels as hk
    counts, lens, heads, kv, dim, page, block = shape
    gen = torch.Generator().manual_seed(1000 + sum(counts) + sum(lens))
    tokens, streams = sum(counts), len(counts)
    keys, values, weights, _, table = make_pool(gen, streams, max(max(lens), 1) + page, kv, page, dim, dtype)
    poison_unused(keys, values, weights, table, lens, page)
    q = (1.5 * torch.randn(tokens, heads, dim, generator=gen)).to(dtype)
    ragged = len(set(counts)) > 1
    starts = starts_of(counts)
    for b, n in enumerate(lens):  # entries behind the slots in use are never read
        table[b, -(-n // page):] = -12345
    lens_t = torch.tensor(lens, dtype=torch.int32)
    out, tol, lse, lse_tol, ww, w_tol = ref.attention(q, keys, values, table, lens_t, starts, None, block, weights, 0.75)
    dev = [t.to(DEV) for t in (q, keys, values, table, lens_t)]
    kw = dict(starts=starts.to(DEV) if ragged else None, causal_block=block)
    got, got_lse = hk.paged_attention(*dev, return_lse=True, **kw)
    ref.assert_within(got, out, tol, "out")
    ref.assert_within(got_lse, lse, lse_tol, "lse")
    w = weights.to(DEV)
    again, again_lse = hk.paged_attention(*dev, weights=w, decay=0.75, return_lse=True, **kw)
    ref.assert_within(again, out, tol, "out with weights")
    ref.assert_within(again_lse, lse, lse_tol, "lse with weights")
    ref.assert_within(w, ww, w_tol, "weights")
    # decay 0 reads no old weight; the log-sum stays inside
    w = torch.full_like(weights, math.nan).to(DEV)
    again = hk.paged_attention(*dev, weights=w, decay=0.0, **kw)
    want0, tol0 = ref.attention(q, keys, values, table, lens_t, starts, None, block, torch.full_like(weights, math.nan), 0.0)[4:]
    ref.assert_within(again, out, tol, "out with weights, decay 0")
    ref.assert_within(w, want0, tol0, "weights, decay 0")


MANY = [  # the same, more than 64 rows a stream; the page table has room for so much that a workgroup takes 128 rows
    ([130], [130], 2, 2, 64, 64, 1),
    ([130], [100], 2, 1, 64, 64, 1),
    ([300], [700], 2, 2, 128, 64, 0),
    ([150], [333], 3, 1, 40, 33, 30),
    ([200, 90, 170], [205, 400, 31], 4, 2, 72, 49, 7),
    ([100, 100], [256, 256], 4, 4, 128, 16, 25),
    ([95], [200], 1, 1, 96, 20, 0),
    ([270], [1], 1, 1, 64, 1, 0),
]


@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("shape", MANY, ids=str)
def test_paged_attention_many_rows(lib, dtype, shape):
    from deltacnn_amd import hip_kernels as hk
    counts, lens, heads, kv, dim, page, block = shape
    gen = torch.Generator().manual_seed(2000 + sum(counts) + sum(lens))
    tokens, streams = sum(counts), len(counts)
    keys, values, weights, _, table = make_pool(gen, streams, max(max(lens), 1) + page, kv, page, dim, dtype)
    poison_unused(keys, values, weights, table, lens, page)
    q = (1.5 * torch.randn(tokens, heads, dim, generator=gen)).to(dtype)
    ragged, starts = len(set(counts)) > 1, starts_of(counts)
    for b, n in enumerate(lens):
        table[b, -(-n // page):] = -12345
    wide = widened(table, page, tokens, heads, kv)
    lens_t = torch.tensor(lens, dtype=torch.int32)
    out, tol, lse, lse_tol, ww, w_tol = ref.attention(q, keys, values, wide, lens_t, starts, None, block, weights, 0.75)
    w = weights.to(DEV)
    got, got_lse = hk.paged_attention(*(t.to(DEV) for t in (q, keys, values, wide, lens_t)), starts=starts.to(DEV) if ragged else None,
                                      causal_block=block, weights=w, decay=0.75, return_lse=True)
    ref.assert_within(got, out, tol, "out")
    ref.assert_within(got_lse, lse, lse_tol, "lse")
    ref.assert_within(w, ww, w_tol, "weights")


@pytest.mark.parametrize("dtype,dim", [(torch.float32, 64), (torch.float16, 64), (torch.bfloat16, 128)], ids=str)
def test_paged_attention_many_rows_in_pieces(lib, dtype, dim):
    """So long a cache that 128 rows of it are joined from several pieces."""
    from deltacnn_amd import hip_kernels as hk
    gen = torch.Generator().manual_seed(31)
    tokens, heads, page, n = 260, 8, 64, 13000
    keys, values, _, _, table = make_pool(gen, 1, n, heads, page, dim, dtype)
    q = (1.5 * torch.randn(tokens, heads, dim, generator=gen)).to(dtype)
    lens_t = torch.tensor([n], dtype=torch.int32)
    out, tol, lse, lse_tol, _, _ = ref.attention(q, keys, values, table, lens_t)
    got, got_lse = hk.paged_attention(*(t.to(DEV) for t in (q, keys, values, table, lens_t)), return_lse=True)
    ref.assert_within(got, out, tol, "out")
    ref.assert_within(got_lse, lse, lse_tol, "lse")


@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("scale", [-0.2, 0.0, 3.0])
@pytest.mark.parametrize("tokens", [2, 70])
def test_paged_attention_scales(lib, dtype, scale, tokens):
    """Negative, zero and large scales, causal and not, rows of a wider buffer as q and out."""
    from deltacnn_amd import hip_kernels as hk
    gen = torch.Generator().manual_seed(31 + tokens)
    heads, kv, dim, page, lens = 4, 2, 48, 32, [100, 75]
    keys, values, weights, _, table = make_pool(gen, 2, 128, kv, page, dim, dtype)
    wide = torch.randn(2 * tokens, heads * dim + 16, generator=gen).to(dtype)
    q = wide[:, :heads * dim].view(2 * tokens, heads, dim)
    lens_t = torch.tensor(lens, dtype=torch.int32)
    for block in (0, 1):
        out, tol, lse, lse_tol, ww, w_tol = ref.attention(q, keys, values, table, lens_t, None, scale, block, weights, 1.0)
        buf = torch.full((2 * tokens, heads * dim + 24), 5.0, dtype=dtype, device=DEV)
        w = weights.to(DEV)
        wd = wide.to(DEV)
        got = hk.paged_attention(wd[:, :heads * dim].view(2 * tokens, heads, dim), keys.to(DEV), values.to(DEV), table.to(DEV),
                                 lens_t.to(DEV), scale=scale, causal_block=block, weights=w,
                                 out=buf[:, 8:8 + heads * dim].view(2 * tokens, heads, dim))
        ref.assert_within(got, out, tol, "out")
        ref.assert_within(w, ww, w_tol, "weights")
        assert bool((buf[:, :8] == 5).all()) and bool((buf[:, 8 + heads * dim:] == 5).all())


@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("tokens,wide", [(3, False), (150, False), (150, True)])
def test_paged_attention_masked_infinities(lib, dtype, tokens, wide):
    """Infinities and NaN in keys and values that a row does not see leave it alone; rows that see
    them get what the definition says."""
    from deltacnn_amd import hip_kernels as hk
    gen = torch.Generator().manual_seed(12)
    dim, page, past = 64, 32, 20
    n = past + tokens
    keys, values, weights, _, table = make_pool(gen, 1, n, 1, page, dim, dtype)
    table = widened(table, page, tokens, 1, 1) if wide else table
    bad = n - max(1, tokens // 2)  # seen by the later rows alone
    pg, off = ref.place(table[0], bad, page)
    values[pg, 0, off, 3], values[pg, 0, off, 40], values[pg, 0, off, 41] = math.nan, math.inf, -math.inf
    q = torch.randn(tokens, 1, dim, generator=gen).to(dtype)
    lens_t = torch.tensor([n], dtype=torch.int32)
    out, tol, lse, lse_tol, _, _ = ref.attention(q, keys, values, table, lens_t, None, None, 1)
    got = hk.paged_attention(q.to(DEV), keys.to(DEV), values.to(DEV), table.to(DEV), lens_t.to(DEV), causal_block=1)
    assert bool(out[:, 0, 3].isnan().any()) and not bool(out[:, 0, 3].isnan().all()) and bool((out[:, 0, 40] == math.inf).any())
    tol = torch.where(out.isfinite(), tol, 0.0)
    ref.assert_within(got, out, tol, "values")
    keys[pg, 0, off, 5] = math.nan  # a key: the rows that see it are NaN, the others are not
    out, tol, lse, lse_tol, _, _ = ref.attention(q, keys, torch.nan_to_num(values, 0, 0, 0), table, lens_t, None, None, 1)
    w = torch.zeros_like(weights).to(DEV)
    got, got_lse = hk.paged_attention(q.to(DEV), keys.to(DEV), torch.nan_to_num(values, 0, 0, 0).to(DEV), table.to(DEV), lens_t.to(DEV),
                                      causal_block=1, weights=w, return_lse=True)
    seen = torch.arange(tokens) + past >= bad
    assert torch.equal(got.isnan().all(2).all(1).cpu(), seen) and torch.equal(got.isnan().any(2).any(1).cpu(), seen)
    ref.assert_within(got[~seen.to(DEV)], out[~seen], tol[~seen], "rows that do not see the key")
    ref.assert_within(got_lse, lse, torch.where(lse.isfinite(), lse_tol, 0.0), "lse")


@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("tokens,wide", [(1, False), (3, False), (70, False), (70, True)])
@pytest.mark.parametrize("block", [0, 1])
def test_paged_attention_visible_infinity(lib, dtype, tokens, wide, block):
    """A key that gives every row a score of -inf: as if the slot were not there, and no weight for it."""
    from deltacnn_amd import hip_kernels as hk
    gen = torch.Generator().manual_seed(15)
    dim, page, n, bad = 64, 32, 400, 127
    keys, values, weights, _, table = make_pool(gen, 1, n, 1, page, dim, dtype)
    table = widened(table, page, tokens, 2, 1) if wide else table
    q = torch.randn(tokens, 2, dim, generator=gen).to(dtype)
    q[:, :, 0] = q[:, :, 0].abs() + 0.5
    lens_t = torch.tensor([n], dtype=torch.int32)
    pg, off = ref.place(table[0], bad, page)
    keys[pg, 0, off] = 0
    keys[pg, 0, off, 0] = -60000.0 / 8  # a score below -400 in the oracle, whose probability is below 2^-500
    out, tol, lse, lse_tol, ww, w_tol = ref.attention(q, keys, values, table, lens_t, None, None, block, weights, 0.5)
    small = keys.clone()
    small[pg, 0, off, 0] = 0  # the bounds: of the scores that count
    tol, lse_tol, w_tol = (ref.attention(q, small, values, table, lens_t, None, None, block, weights, 0.5)[i] for i in (1, 3, 5))
    keys[pg, 0, off, 0] = -math.inf
    w = weights.to(DEV)
    got, got_lse = hk.paged_attention(q.to(DEV), keys.to(DEV), values.to(DEV), table.to(DEV), lens_t.to(DEV), causal_block=block, weights=w,
                                      decay=0.5, return_lse=True)
    assert float(w[pg, 0, off]) == 0.5 * float(weights[pg, 0, off])
    ref.assert_within(got_lse, lse, lse_tol, "lse")
    ref.assert_within(w, ww, w_tol, "weights")
    # (a bound with the slot's value in it is the larger one; both are within half a percent of sum p |v|)
    ref.assert_within(got, out, 1.01 * tol, "out")


@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("tokens,page", [(2, 32), (2, 20), (80, 64), (80, 20), (2, 48), (80, 48), (2, 16), (80, 16)])
def test_paged_attention_lost_page_and_rows_behind(lib, dtype, tokens, page, wide):
    """A page outside the pool makes its own stream NaN and no other; rows behind the last stream stay."""
    from deltacnn_amd import hip_kernels as hk
    gen = torch.Generator().manual_seed(3)
    dim, lens = 32, [90, 130, 41]
    keys, values, weights, _, table = make_pool(gen, 3, 140, 1, page, dim, dtype)
    table[1, 1] = keys.shape[0] if page > 20 else -1
    table = widened(table, page, 3 * tokens, 2, 1) if wide else table
    counts = [tokens, tokens, tokens - 1]
    starts = starts_of(counts)
    total = sum(counts) + 4
    q = torch.randn(total, 2, dim, generator=gen).to(dtype)
    lens_t = torch.tensor(lens, dtype=torch.int32)
    safe = table.clone()
    safe[1] = safe[0]
    out, tol, lse, _, _, _ = ref.attention(q[:sum(counts)], keys, values, safe, lens_t, starts, None, 0)
    buf = torch.full((total, 2, dim), 9.0, dtype=dtype, device=DEV)
    w = weights.to(DEV)
    got = hk.paged_attention(q.to(DEV), keys.to(DEV), values.to(DEV), table.to(DEV), lens_t.to(DEV), starts=starts.to(DEV), out=buf, weights=w)
    second = slice(counts[0], 2 * tokens)
    assert bool(got[second].isnan().all()) and bool((got[sum(counts):] == 9).all())
    for part in (slice(0, tokens), slice(2 * tokens, sum(counts))):
        ref.assert_within(got[part], out[part], tol[part], "other streams")
    touched = torch.zeros(keys.shape[0], dtype=torch.bool)
    for b in (0, 1, 2):
        for i in range(-(-lens[b] // page)):
            if 0 <= int(table[b, i]) < keys.shape[0]:
                touched[int(table[b, i])] = True
    assert torch.equal(w.cpu()[~touched], weights[~touched])


# ---- cache_slots ----

SLOTS = [  # counts, lens, budget, kv_heads, page, protect
    ([1], [1], 1, 1, 1, None), ([5], [20], 20, 2, 7, None), ([5], [20], 22, 2, 7, 6), ([5], [20], 64, 1, 64, 6),
    ([3, 0, 7], [50, 9, 1], 50, 3, 16, 5), ([40], [40], 40, 2, 49, 3), ([9], [64], 64, 1, 64, 0),  # all protected
    ([200], [1000], 1000, 2, 100, 8), ([64, 64], [2500, 2499], 2500, 1, 64, 7), ([30], [10], 20, 1, 30, None),
    ([12, 12], [100, 3], 40, 1, 10, 4),       # one stream is over its budget already: it does not shrink
    ([700], [9000], 9000, 1, 64, 7), ([50], [20000], 20000, 1, 128, 8),    # several slots a thread
    ([3000, 10], [40000, 33000], 40000, 1, 64, 6), ([2100], [70000], 70000, 2, 100, 1),  # cut into pieces
]


@pytest.mark.parametrize("kind", ["random", "ties", "odd"])
@pytest.mark.parametrize("shape", SLOTS, ids=str)
def test_cache_slots(lib, kind, shape):
    from deltacnn_amd import hip_kernels as hk
    counts, lens, budget, kv, page, protect = shape
    gen = torch.Generator().manual_seed(9 + sum(counts))
    streams = len(counts)
    _, _, weights, stamps, table = make_pool(gen, streams, max(max(lens), budget), kv, page, 8, torch.float16)
    if kind == "ties":
        weights = torch.randint(0, 3, weights.shape, generator=gen).float()
    if kind == "odd":
        pick = torch.randint(0, 7, weights.shape, generator=gen)
        special = torch.tensor([0.0, -0.0, math.nan, math.inf, -math.inf, 1e-42, -3.0])
        weights = torch.where(torch.rand(weights.shape, generator=gen) < 0.6, special[pick], weights)
        if streams > 1:
            table[0, 0] = -1
    starts = starts_of(counts)
    lens_t = torch.tensor(lens, dtype=torch.int32)
    keep = None if protect is None else torch.full((streams,), protect, dtype=torch.int32)
    st = None if protect is None else stamps
    total = sum(counts) + (2 if len(set(counts)) > 1 else 0)
    want, new = ref.slots(weights, table, lens_t, total, budget, starts, st, keep)
    on = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    got, got_new = hk.cache_slots(on(weights), on(table), on(lens_t), total, budget, starts=on(starts) if len(set(counts)) > 1 else None,
                                  stamps=on(st), keep_from=on(keep))
    n = sum(counts)
    assert torch.equal(got.cpu()[:, :n], want[:, :n]) and torch.equal(got_new.cpu(), new)


# ---- the operators together ----

class PlainFrames:
    """The layer in 64 bits, token by token lists instead of slots: what a stream holds, per kv head."""

    def __init__(self, layer, shape):
        self.l, self.shape = layer, shape
        self.kept = [[[] for _ in range(layer.kv_heads)] for _ in range(shape[0])]  # lists by slot: [key, value, weight, stamp]
        self.t, self.gap = 0, math.inf  # gap: between the last weight that went and the first that stayed

    def frame(self, x):
        l, (b, c, h, w) = self.l, self.shape
        n, dim = h * w, l.head_dim
        fused = x.permute(0, 2, 3, 1).reshape(b * n, c).double() @ l.qkv.weight.double().cpu().T + l.qkv.bias.double().cpu()
        q, k, v = fused.split([l.heads * dim, l.kv_heads * dim, l.kv_heads * dim], 1)
        grid = torch.stack(torch.meshgrid(torch.arange(b) * 0 + self.t, torch.arange(h), torch.arange(w), indexing="ij"), -1).reshape(-1, 3)
        from deltacnn_amd import hip_kernels as hk
        freq = hk.rotary_frequencies(l.sections, l.base)
        q = ref.rotary(q.reshape(b * n, l.heads, dim), grid, freq, l.sections, False)[0]
        k = ref.rotary(k.reshape(b * n, l.kv_heads, dim), grid, freq, l.sections, False)[0]
        v = v.reshape(b * n, l.kv_heads, dim)
        out = torch.zeros(b * n, l.heads, dim, dtype=torch.float64)
        group = l.heads // l.kv_heads
        for s in range(b):
            for g in range(l.kv_heads):
                cells = self.kept[s][g]
                rows = range(s * n, (s + 1) * n)
                e = max(0, len(cells) + n - l.frames * n)
                order = sorted(range(len(cells)), key=lambda i: (cells[i][3] >= self.t - l.keep_frames + 1, cells[i][2], i))
                freed = sorted(order[:e])
                if 0 < e < len(order) and (cells[order[e - 1]][3] >= self.t - l.keep_frames + 1) == (cells[order[e]][3] >= self.t - l.keep_frames + 1):
                    self.gap = min(self.gap, cells[order[e]][2] - cells[order[e - 1]][2])
                for j, r in enumerate(rows):
                    cell = [k[r, g], v[r, g], 0.0, self.t]
                    if j < e:
                        cells[freed[j]] = cell
                    else:
                        cells.append(cell)
                kk, vv = torch.stack([x[0] for x in cells]), torch.stack([x[1] for x in cells])
                got = torch.zeros(len(cells), dtype=torch.float64)
                for r in rows:
                    for hd in range(g * group, (g + 1) * group):
                        p = torch.softmax(kk @ q[r, hd] * dim ** -0.5, 0)
                        out[r, hd] = p @ vv
                        got += p
                for i, cell in enumerate(cells):
                    cell[2] = l.decay * cell[2] + float(got[i])
        self.t += 1
        y = out.reshape(b * n, -1) @ l.proj.weight.double().cpu().T + l.proj.bias.double().cpu()
        return y.view(b, h, w, c).permute(0, 3, 1, 2)


def _layer(dtype, frames=3, kv=2):
    from deltacnn_amd.sparse_layers import DCFrameAttention
    torch.manual_seed(4)
    return DCFrameAttention(48, 4, kv_heads=kv, head_dim=24, frames=frames, keep_frames=1, decay=0.5, page_size=16).eval().to(DEV).to(dtype)


def test_layer_follows_its_definition(lib):
    """fp32, two streams, five frames of which three fit: slots, positions, weights and eviction as a whole.

    The layer's numbers are sums of at most 48 (projections) and 60 (slots) terms of magnitude about 1 in
    fp32 behind two projections: 10 (48 + 60) w relative to outputs below 1; weights that decide an eviction
    have to differ by more than twice that, or the choice would be the rounding's."""
    layer = _layer(torch.float32)
    shape = (2, 48, 4, 5)
    plain = PlainFrames(layer, shape)
    gen = torch.Generator().manual_seed(8)
    with torch.no_grad():
        for t in range(5):
            x = torch.randn(shape, generator=gen)
            want = plain.frame(x)
            got = layer(x.to(DEV).contiguous(memory_format=torch.channels_last))
            assert got.is_contiguous(memory_format=torch.channels_last)
            assert float((got.double().cpu() - want).abs().max()) < 10 * 108 * ref.W, f"frame {t}"
            s = layer._state
            assert s["lens"].tolist() == [min(t + 1, 3) * 20] * 2
            for b in range(2):
                for h in range(2):
                    cells = plain.kept[b][h]
                    stamps = ref.gather(s["stamps"].cpu()[..., None], s["table"].cpu()[b], len(cells), h, 16)[:, 0]
                    assert stamps.tolist() == [c[3] for c in cells], f"frame {t}: other tokens were kept"
    assert 20 * 108 * ref.W < plain.gap < math.inf


@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("size", [(1, 1), (7, 7), (12, 9)], ids=str)
def test_layer_replays_from_a_graph(lib, dtype, size):
    """Frames replayed from a captured graph, eager work of another layer in between, equal eager frames
    bit for bit; two graphs of two layers do not disturb each other."""
    from deltacnn_amd.graph import FrameGraph
    shape = (2, 48) + size
    gen = torch.Generator().manual_seed(21)
    video = [torch.randn(shape, generator=gen).to(dtype).to(DEV).contiguous(memory_format=torch.channels_last) for _ in range(8)]
    eager, first, second = _layer(dtype), _layer(dtype), _layer(dtype)
    with torch.no_grad():
        wanted = [eager(x).clone() for x in video]
        for layer in (first, second):
            assert torch.equal(layer(video[0]), wanted[0])
        graphs = [FrameGraph(first, video[0]), FrameGraph(second, video[0])]
        other = _layer(dtype)
        for t in range(1, 8):
            a, b = graphs[0](video[t]).clone(), graphs[1](video[t]).clone()
            other(video[t])
            torch.cuda.synchronize()
            assert torch.equal(a, wanted[t]) and torch.equal(b, wanted[t]), f"frame {t}"


def test_layer_starts_anew(lib):
    layer = _layer(torch.float16)
    x = torch.randn(1, 48, 3, 3, device=DEV).half().contiguous(memory_format=torch.channels_last)
    with torch.no_grad():
        a = layer(x).clone()
        layer(x)
        layer.reset()
        assert torch.equal(layer(x), a)
        layer(torch.cat([x, x]))                    # another number of streams: another state
        assert layer._state["lens"].tolist() == [9, 9]
        with pytest.raises(TypeError):
            layer((x, None))
    from deltacnn_amd import _lib
    with pytest.raises(_lib.DeltaCNNError, match="gradient"):
        layer(x)


def test_numbers_beyond_32_bits_are_refused(lib):
    from deltacnn_amd import _lib
    from deltacnn_amd import hip_kernels as hk
    pool, table, lens = torch.zeros(2, 1, 8, 16, device=DEV), torch.zeros(1, 2, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    q = torch.zeros(1, 1, 16, device=DEV)
    for call in (lambda: hk.paged_attention(q, pool, pool, table, lens, causal_block=1 << 32),
                 lambda: hk.cache_slots(pool[..., 0].contiguous(), table, lens, (1 << 32) + 1, 8),
                 lambda: hk.cache_slots(pool[..., 0].contiguous(), table, lens, 1, (1 << 32) + 8)):
        with pytest.raises(_lib.DeltaCNNError, match="32 bits"):
            call()


def test_layer_under_the_tracer(lib):
    from deltacnn_amd import hip_kernels as hk
    from deltacnn_amd.trace import Tracer
    layer = _layer(torch.float16)
    x = torch.randn(2, 48, 4, 4, device=DEV).half().contiguous(memory_format=torch.channels_last)
    tracer = Tracer()
    with torch.no_grad():
        layer(x)
        hk.set_tracer(tracer)
        try:
            layer(x)
        finally:
            hk.set_tracer(None)
    rows = {r["call"]: r for r in tracer.finish()}
    assert {"cache_slots", "rotary_append", "paged_attention"} <= set(rows)
    assert rows["paged_attention"]["flops"] == 4 * (2 * 16 * 32) * 4 * 24
    assert rows["rotary_append"]["bytes"] == 2 * 32 * 8 * 24 * 2 + 32 * (3 + 2) * 4 + 32 * 2 * 8


def test_operators_on_another_stream(lib):
    """Operands made on one stream, the operators on another that waits for it."""
    from deltacnn_amd import hip_kernels as hk
    gen = torch.Generator().manual_seed(2)
    keys, values, weights, _, table = (t.to(DEV) for t in make_pool(gen, 1, 4000, 2, 64, 64, torch.float16))
    q = torch.randn(60, 4, 64, generator=gen).half().to(DEV)
    lens = torch.tensor([4000], dtype=torch.int32, device=DEV)
    want, w_want = hk.paged_attention(q, keys, values, table, lens), weights.clone()
    hk.paged_attention(q, keys, values, table, lens, weights=w_want)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    late = torch.zeros_like(q)
    w = weights.clone()
    big = torch.randn(4096, 4096, device=DEV)
    for _ in range(4):
        big = big @ big * 1e-2
    late.copy_(q)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = hk.paged_attention(late, keys, values, table, lens, weights=w)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want) and torch.equal(w, w_want)


def test_results_do_not_change_from_run_to_run(lib):
    from deltacnn_amd import hip_kernels as hk
    gen = torch.Generator().manual_seed(6)
    keys, values, weights, stamps, table = (t.to(DEV) for t in make_pool(gen, 2, 9000, 2, 64, 128, torch.bfloat16))
    lens = torch.tensor([9000, 7777], dtype=torch.int32, device=DEV)
    for tokens in (2, 2 * 200):
        q = torch.randn(tokens, 8, 128, generator=gen).bfloat16().to(DEV)
        seen = []
        for _ in range(4):
            w = weights.clone()
            seen.append((hk.paged_attention(q, keys, values, table, lens, weights=w, decay=0.5), w))
        assert all(torch.equal(a, seen[0][0]) and torch.equal(b, seen[0][1]) for a, b in seen)


@pytest.mark.parametrize("page", [64, 60])
def test_pool_beyond_32_bit_offsets(lib, page):
    """The last pages of a pool of more than 2^31 elements: the same results as a small pool's."""
    from deltacnn_amd import hip_kernels as hk
    dim, kv, n = 256, 2, 4 * page
    pages = (1 << 31) // (kv * page * dim) + 40
    dtype = torch.float16
    gen = torch.Generator().manual_seed(1)
    small_k, small_v = (torch.randn(4, kv, page, dim, generator=gen).to(dtype).to(DEV) for _ in range(2))
    keys = torch.zeros(pages, kv, page, dim, dtype=dtype, device=DEV)
    values = torch.zeros_like(keys)
    keys[-4:], values[-4:] = small_k, small_v
    far = torch.arange(pages - 4, pages, dtype=torch.int32, device=DEV)[None]
    near = torch.arange(4, dtype=torch.int32, device=DEV)[None]
    lens = torch.tensor([n], dtype=torch.int32, device=DEV)
    for tokens in (1, 70):
        q = torch.randn(tokens, 2, dim, generator=gen).to(dtype).to(DEV)
        w_far, w_near = torch.zeros(pages, kv, page, device=DEV), torch.zeros(4, kv, page, device=DEV)
        a = hk.paged_attention(q, keys, values, far, lens, weights=w_far)
        b = hk.paged_attention(q, small_k, small_v, near, lens, weights=w_near)
        assert torch.equal(a, b) and torch.equal(w_far[-4:], w_near)
    # and writing there
    k = torch.randn(5, kv, dim, generator=gen).to(dtype).to(DEV)
    pos = torch.arange(5, dtype=torch.int32, device=DEV)[:, None].contiguous()
    slots = torch.arange(n - 5, n, dtype=torch.int32, device=DEV).expand(kv, 5).contiguous()
    freq = hk.rotary_frequencies((dim,), device=DEV)
    hk.rotary_append(k, k, k, pos, freq, (dim,), keys, values, far, slots)
    assert torch.equal(values[-1, :, page - 5:], k.transpose(0, 1)) and torch.equal(keys[:-4].view(torch.int16).amax(), keys.new_zeros((), dtype=torch.int16))
