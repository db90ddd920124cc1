"""Paged serving operators (append, ragged chunk attention, key weights, eviction)
against plain float64 implementations.

Tolerances, from the formulas:
  * a score s = scale q.k is a float32 sum of D exact products: the error of such a sum
    is about sqrt(D) roundings of its largest partial sum, so |ds| <= DS =
    4 sqrt(D) 2^-24 scale max sum|q_d k_d|;
  * outputs: p is rounded to the 16-bit type before P V (relative U = the type's unit
    roundoff: 2^-8 for bfloat16, 2^-11 for float16, 2^-24 for float32) and so is the result; a score error moves p by at most
    2 DS dp/ds.  |do| <= 2 U sum p|v| + 2 DS sum g |v| + 1e-6 max|v|;
  * key weights stay in float32: |dw| <= 2 DS sum g + 1e-6 w, summed over the rows,
with g = dp/ds up to the threshold's own error: p (softmax1), 1[z > tau - 2 DS]
(sparsemax), sqrt(p) + DS (entmax15).
"""

import math

import numpy as np
import pytest
import torch

import oracle
from hf_attention_normalizers_b200 import serving

pytestmark = pytest.mark.gpu

NORMS = ("softmax1", "sparsemax", "entmax15")
# half the spacing of 1 + eps: significands of 24, 11 and 8 bits
UNIT = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.float16, torch.bfloat16)}


class Batch:
    """A paged cache with a ragged batch on it.  Slots that belong to no key hold NaN."""

    def __init__(self, new, lens, *, hkv=2, group=4, dim=128, page=32, dtype=torch.bfloat16, seed=0, gain=1.0,
                 interleave=False, extra_blocks=1, spare=2, stale=float("nan")):
        g = torch.Generator().manual_seed(seed)
        self.new, self.lens, self.hkv, self.group, self.dim, self.page, self.dtype = new, lens, hkv, group, dim, page, dtype
        pages = [max(1, -(-c // page)) for c in lens]
        order = torch.randperm(sum(pages) + spare, generator=g)
        self.table = torch.full((len(lens), max(pages) + extra_blocks), -1, dtype=torch.int32)
        self.rows = []
        at = 0
        for b, (n, c) in enumerate(zip(pages, lens)):
            self.table[b, :n] = order[at:at + n]
            at += n
            pos = torch.arange(c)
            self.rows.append(self.table[b].long()[pos // page] * page + pos % page)
        slots = (sum(pages) + spare) * page
        kc = torch.full((slots, hkv, dim), stale)
        vc = torch.full((slots, hkv, dim), stale)
        for r in self.rows:
            kc[r] = torch.randn(len(r), hkv, dim, generator=g)
            vc[r] = torch.randn(len(r), hkv, dim, generator=g)
        total = sum(new)
        self.query = (torch.randn(total, hkv * group, dim, generator=g) * gain).to(dtype)
        self.key_cache, self.value_cache = kc.to(dtype), vc.to(dtype)
        self.weights = torch.rand(hkv, slots, generator=g)
        self.cu = torch.tensor([0] + list(np.cumsum(new)), dtype=torch.int32)
        self.seq = torch.tensor(lens, dtype=torch.int32)
        dev = "cuda"
        self.d_query, self.d_table, self.d_cu, self.d_seq = (t.to(dev) for t in (self.query, self.table, self.cu, self.seq))
        self.d_weights = self.weights.to(dev)
        if interleave:  # K and V of a token side by side in one allocation
            both = torch.stack((self.key_cache, self.value_cache), 1).to(dev)
            self.d_key, self.d_value = both[:, 0], both[:, 1]
        else:
            self.d_key, self.d_value = self.key_cache.to(dev), self.value_cache.to(dev)

    def chunk(self, norm, **kw):
        kw.setdefault("max_seqlen_q", max(self.new))
        kw.setdefault("max_seqlen_k", max(self.lens))
        return serving.paged_chunk_attention(self.d_query, self.d_key, self.d_value, self.d_table, self.d_cu, self.d_seq,
                                             self.page, normalizer=norm, **kw)

    def expected(self, norm, causal=True, scale=None):
        """Outputs, their tolerance, added key weights and their tolerance (float64)."""
        scale = self.dim ** -0.5 if scale is None else scale
        u = UNIT[self.dtype]
        out = np.zeros(self.query.shape)
        tol = np.zeros(self.query.shape)
        add, add_tol = np.zeros(self.weights.shape), np.zeros(self.weights.shape)
        q_all, kc, vc = self.query.double().numpy(), self.key_cache.double().numpy(), self.value_cache.double().numpy()
        for b, (n, c) in enumerate(zip(self.new, self.lens)):
            rows = self.rows[b].numpy()
            for h in range(self.query.shape[1]):
                kvh = h // self.group
                k, v = kc[rows, kvh], vc[rows, kvh]
                for i in range(n):
                    t = int(self.cu[b]) + i
                    see = min(c, c - n + i + 1) if causal else c
                    if see <= 0:
                        continue
                    q = q_all[t, h]
                    x = scale * (k[:see] @ q)
                    p = oracle.normalize(norm, x[None])[0]
                    ds = 4 * math.sqrt(self.dim) * 2.0 ** -24 * abs(scale) * (np.abs(k[:see]) @ np.abs(q)).max()
                    if norm == "softmax1":
                        g = p
                    elif norm == "entmax15":
                        g = np.sqrt(p) + ds
                    else:
                        tau = x[p > 0].min() - p[p > 0].min()
                        g = (x > tau - 2 * ds).astype(np.float64)
                    av = np.abs(v[:see])
                    out[t, h] = p @ v[:see]
                    tol[t, h] = 2 * u * (p @ av) + 2 * ds * (g @ av) + 1e-6 * av.max()
                    add[kvh, rows[:see]] += p
                    add_tol[kvh, rows[:see]] += 2 * ds * g + 1e-6 * p
        return out, tol, add, add_tol


def _check(actual, expected, tol, what):
    a = actual.detach().double().cpu().numpy()
    assert np.isfinite(a).all(), f"{what}: non-finite values"
    over = np.abs(a - expected) - tol
    assert over.max() <= 0, f"{what}: {over.max():.3e} over the tolerance, error {np.abs(a - expected).max():.3e}"


def _chunk_case(batch, norm, causal=True, scale=None, **kw):
    before = batch.weights.double().numpy()
    out = batch.chunk(norm, is_causal=causal, scale=scale, key_weights=batch.d_weights, **kw)
    want, tol, add, add_tol = batch.expected(norm, causal, scale)
    _check(out, want, tol, f"{norm}/out")
    # the accumulators themselves are float32
    _check(batch.d_weights, before + add, add_tol + 1e-6 * (before + add), f"{norm}/weights")
    assert serving.device_status() == 0


SHAPES = [
    # new, lens, layout
    ([1], [1], {}),
    ([1, 1, 1], [1, 33, 200], {}),
    ([5], [5], dict(group=1)),
    ([7, 0, 130], [40, 9, 131], {}),
    ([3, 65, 1, 0], [3, 300, 257, 0], dict(group=5, hkv=1)),
    ([64, 33], [64, 100], dict(group=7, hkv=2, dim=64)),
    ([129], [700], dict(group=2, hkv=1, page=16)),
    ([20, 1], [150, 1000], dict(group=8, hkv=2, dim=64, page=64)),
    ([40], [383], dict(page=128)),
    ([17, 9], [50, 270], dict(page=256, hkv=1)),
    ([9, 4], [61, 44], dict(page=24, hkv=1)),
    ([6, 2], [30, 77], dict(page=8, hkv=1)),
    ([12], [45], dict(page=5, hkv=1)),
    ([10, 3], [33, 90], dict(dim=40, hkv=1)),
    ([3], [70], dict(group=48, hkv=1)),
    ([2], [50], dict(group=160, hkv=1, dim=64)),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("norm", NORMS)
@pytest.mark.parametrize("case", range(len(SHAPES)))
def test_chunk_attention_and_key_weights(case, norm, dtype):
    new, lens, kw = SHAPES[case]
    _chunk_case(Batch(new, lens, dtype=dtype, seed=case, gain=2.0, **kw), norm)


@pytest.mark.parametrize("norm", NORMS)
def test_chunk_without_causal_mask(norm):
    _chunk_case(Batch([33, 4], [150, 40], seed=3), norm, causal=False)


@pytest.mark.parametrize("norm", NORMS)
@pytest.mark.parametrize("scale", [0.0, -0.05, 0.6])
def test_chunk_scales(norm, scale):
    """Equal scores (every key in the sparse support), negative and large scales."""
    _chunk_case(Batch([20, 1], [500, 300], seed=4), norm, scale=scale)


@pytest.mark.parametrize("norm", NORMS)
def test_rows_without_a_visible_key_are_zero(norm):
    """More new tokens than keys: the first rows see nothing."""
    b = Batch([9, 140], [4, 130], seed=5)
    _chunk_case(b, norm)
    out = b.chunk(norm)
    assert (out[:5] == 0).all() and (out[9:19] == 0).all() and out[5:9].abs().amax() > 0


@pytest.mark.parametrize("norm", NORMS)
def test_interleaved_cache_strided_query_and_no_hints(norm):
    b = Batch([30, 1, 70], [90, 257, 400], seed=6, interleave=True)
    wide = torch.zeros(b.query.shape[0], b.query.shape[1], 3 * b.dim, dtype=b.dtype, device="cuda")
    wide[..., b.dim:2 * b.dim] = b.d_query
    b.d_query = wide[..., b.dim:2 * b.dim]
    b.d_table, b.d_cu, b.d_seq = b.d_table.long(), b.d_cu.long(), b.d_seq.long()
    _chunk_case(b, norm, max_seqlen_q=None, max_seqlen_k=None)


@pytest.mark.parametrize("norm", NORMS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_unaligned_query_view(norm, dtype):
    """A query view whose rows start off a 16-byte boundary."""
    b = Batch([30, 5], [90, 41], seed=7, dtype=dtype)
    wide = torch.zeros(b.query.shape[0], b.query.shape[1], b.dim + 3, dtype=b.dtype, device="cuda")
    wide[..., 1:b.dim + 1] = b.d_query
    b.d_query = wide[..., 1:b.dim + 1]
    _chunk_case(b, norm)


@pytest.mark.parametrize("norm", NORMS)
def test_long_context_few_rows(norm):
    """The key axis is split between thread blocks when there are few rows."""
    _chunk_case(Batch([3, 1], [9001, 4100], seed=8, hkv=1, gain=2.0), norm)


@pytest.mark.parametrize("norm", NORMS)
def test_decode_batch(norm):
    _chunk_case(Batch([1] * 5, [700, 1, 32, 1025, 64], seed=9, gain=2.0), norm)


@pytest.mark.parametrize("norm", NORMS)
def test_infinities_and_nan_outside_the_length(norm):
    for stale in (float("inf"), -float("inf"), float("nan")):
        _chunk_case(Batch([40, 2], [100, 70], seed=10, stale=stale), norm)


def test_peaked_and_flat_rows_share_a_tile():
    """Rows of one tile whose scores differ a lot in size: one key with everything beside even rows."""
    for norm in NORMS:
        b = Batch([32], [600], seed=11, hkv=1)
        b.query[::2] *= 12.0
        b.query[1::2] *= 0.01
        b.d_query = b.query.cuda()
        _chunk_case(b, norm)


@pytest.mark.parametrize("new", [[1, 1], [2, 5], [70, 40]])
@pytest.mark.parametrize("norm", NORMS)
def test_scores_that_grow_along_the_keys(norm, new):
    """Row maxima that rise by far more than 2^8 from one key tile to the next, and from one part of the keys to another."""
    b = Batch(new, [900, 3000], seed=18, hkv=1)
    for r in b.rows:
        b.key_cache[r] *= torch.linspace(0.1, 25.0, len(r)).to(b.dtype)[:, None, None]
    b.d_key = b.key_cache.cuda()
    _chunk_case(b, norm)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("group,new", [(1, [1, 32, 0, 7]), (8, [4, 1, 2]), (3, [5, 1]), (32, [1, 1]), (5, [3, 1, 0, 1])])
def test_few_rows(group, new, dim):
    lens = [513, 100, 1300, 129, 64][:len(new)]
    _chunk_case(Batch(new, lens, seed=19, group=group, hkv=2, dim=dim, gain=2.0), "softmax1")


def test_wrong_hint_of_the_longest_chunk():
    """A hint smaller than a sequence's chunk only sets the tile size."""
    _chunk_case(Batch([40, 3], [300, 130], seed=20), "softmax1", max_seqlen_q=2)


def test_same_bits_on_every_run():
    for norm in NORMS:
        outs = []
        for _ in range(2):
            b = Batch([100, 1, 30], [900, 3000, 300], seed=12)
            outs.append((b.chunk(norm, key_weights=b.d_weights), b.d_weights))
        assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])


@pytest.mark.parametrize("norm", NORMS)
def test_shared_pages_add_for_every_sequence(norm):
    """Two sequences whose prefix is the same page: both add to its accumulators."""
    b = Batch([4, 6], [64, 70], seed=13, hkv=1)
    b.table[1, 0] = b.table[0, 0]
    b.rows[1] = b.table[1].long()[torch.arange(70) // 32] * 32 + torch.arange(70) % 32
    b.d_table = b.table.cuda()
    _chunk_case(b, norm)


def test_on_another_stream():
    b = Batch([50, 3], [200, 90], seed=14)
    ref = b.chunk("softmax1")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = b.chunk("softmax1")
    side.synchronize()
    assert torch.equal(out, ref)


@pytest.mark.parametrize("norm", NORMS)
@pytest.mark.parametrize("new", [[1, 1, 1], [70, 1, 200]])
def test_in_a_cuda_graph(norm, new):
    b = Batch(new, [500, 40, 1200], seed=15)
    eager = b.chunk(norm, key_weights=b.d_weights)
    w = b.weights.cuda()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = b.chunk(norm, key_weights=w)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, eager) and torch.equal(w, b.d_weights)


def test_traced_by_compile():
    b = Batch([5, 1], [80, 40], seed=16)

    def step(q, kc, vc, w):
        return serving.paged_chunk_attention(q, kc, vc, b.d_table, b.d_cu, b.d_seq, b.page, "entmax15", key_weights=w,
                                             max_seqlen_q=5, max_seqlen_k=80) * 2

    w = b.weights.cuda()
    got = torch.compile(step, fullgraph=True, backend="aot_eager")(b.d_query, b.d_key, b.d_value, w)
    want = step(b.d_query, b.d_key, b.d_value, b.d_weights)
    assert torch.equal(got, want) and torch.equal(w, b.d_weights)


def test_bad_page_and_length_are_recorded():
    """A page id outside the cache reads as zeros, a length past the hint is clamped; both set the status word."""
    for norm in NORMS:
        b = Batch([20, 3], [100, 50], seed=17)
        serving.device_status()
        b.d_table[0, 1] = 10 ** 6
        out = b.chunk(norm)
        assert torch.isfinite(out).all() and serving.device_status() == 1 and serving.device_status() == 0
        b.d_table.copy_(b.table)
        b.chunk(norm, max_seqlen_k=90)
        assert serving.device_status() == 3


def _stale_results(b):
    """Leave NaN in the allocator's blocks that the next call's output and statistics will take."""
    junk = [torch.full_like(b.d_query, float("nan")) for _ in range(3)]
    junk += [torch.full((2, b.query.shape[1], b.query.shape[0]), float("nan"), device="cuda") for _ in range(3)]
    del junk


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("group,new", [(4, [1, 1]), (8, [4, 1])])
def test_decoding_rounds_the_result_only(group, new, dim, dtype):
    """Few rows: P goes into P V as two 16-bit parts, whose sum is off by U^2 (and by float16's least step 2^-25 of the largest)."""
    b = Batch(new, [5000, 700], seed=57, group=group, hkv=2, dim=dim, dtype=dtype)
    out = b.chunk("softmax1")
    want, loose, _, _ = b.expected("softmax1")
    u = UNIT[dtype]
    q_all, kc, vc = b.query.double().numpy(), b.key_cache.double().numpy(), b.value_cache.double().numpy()
    tol = np.zeros(want.shape)
    for s, (n, c) in enumerate(zip(b.new, b.lens)):
        rows = b.rows[s].numpy()
        for h in range(want.shape[1]):
            k, v = kc[rows, h // group], np.abs(vc[rows, h // group])
            for i in range(n):
                t, see = int(b.cu[s]) + i, c - n + i + 1
                x = dim ** -0.5 * (k[:see] @ q_all[t, h])
                p = np.exp(x) / (1.0 + np.exp(x).sum())
                ds = 4 * math.sqrt(dim) * 2.0 ** -24 * dim ** -0.5 * (np.abs(k[:see]) @ np.abs(q_all[t, h])).max()
                step = 2.0 ** -25 * max(p.max(), 0.0) if dtype is torch.float16 else 0.0
                # (the float32 sums of see products: 1e-6 of the largest value, as in expected())
                tol[t, h] = 1.01 * u * np.abs(want[t, h]) + (u * u + 2 * ds) * (p @ v[:see]) + step * v[:see].sum(0) \
                    + 1e-6 * v[:see].max()
    _check(out, want, tol, "out")


@pytest.mark.parametrize("hint", [0, 2])
@pytest.mark.parametrize("norm", NORMS)
@pytest.mark.parametrize("kw", [dict(), dict(dtype=torch.float32), dict(dim=40), dict(page=5), dict(group=48, hkv=1),
                                dict(group=160, hkv=1, dim=64)])
def test_low_hint_of_the_longest_chunk(kw, norm, hint):
    """Rows past the hint are computed all the same, by every kernel."""
    b = Batch([40, 3], [300, 130], seed=53, gain=2.0, **kw)
    _stale_results(b)
    _chunk_case(b, norm, max_seqlen_q=hint)


@pytest.mark.parametrize("norm", NORMS)
@pytest.mark.parametrize("kw", [dict(), dict(dtype=torch.float32), dict(dim=64, dtype=torch.float16, group=3)])
@pytest.mark.parametrize("new,lens", [([1, 2], [200, 300]), ([60, 70], [200, 300]), ([0, 0], [20, 7])])
def test_rows_of_no_sequence_are_zero(new, lens, kw, norm):
    """A padded batch: packed rows before the first offset and past the last one."""
    b = Batch(new, lens, seed=55, gain=2.0, **kw)
    want, tol, add, add_tol = b.expected(norm)
    front, back, n = 5, 37, sum(new)
    query = torch.full((front + n + back, *b.query.shape[1:]), 3.0, dtype=b.dtype, device="cuda")
    query[front:front + n] = b.d_query
    b.d_query, b.query, b.d_cu = query, query, b.d_cu + front
    _stale_results(b)
    out = b.chunk(norm, key_weights=b.d_weights)
    assert (out[:front] == 0).all() and (out[front + n:] == 0).all()
    _check(out[front:front + n], want, tol, norm) if n else None
    before = b.weights.double().numpy()
    _check(b.d_weights, before + add, add_tol + 1e-6 * (before + add), f"{norm}/weights")
    assert serving.device_status() == 0


def _low_scores(b, profile):
    """Scores of the given profile (natural units, along the keys) for every row, values that do not cancel."""
    b.query.zero_()
    b.query[..., 0] = 4.0
    for r in b.rows:
        b.key_cache[r] = torch.randn(b.key_cache[r].shape, generator=torch.Generator().manual_seed(7)).to(b.dtype)
        b.key_cache[r, :, 0] = (profile(len(r)) / (4.0 * b.dim ** -0.5)).to(b.dtype)[:, None]
        b.value_cache[r] = b.value_cache[r].abs()
    b.d_query, b.d_key, b.d_value = b.query.cuda(), b.key_cache.cuda(), b.value_cache.cuda()


LOW_SCORES = {
    "even": lambda n: torch.full((n,), -17.0),
    "range": lambda n: -18.0 + 6.0 * torch.rand(n, generator=torch.Generator().manual_seed(8)),
    "lower": lambda n: torch.full((n,), -22.0),
    "lowest": lambda n: torch.full((n,), -90.0),
    "rising": lambda n: torch.linspace(-24.0, 9.0, n),
    "falling": lambda n: torch.linspace(9.0, -24.0, n),
    "one high key": lambda n: torch.where(torch.arange(n) == n - 70, -3.0, -17.0),
}


@pytest.mark.parametrize("profile", LOW_SCORES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new", [[1, 3], [70, 2]])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_rows_that_attend_to_almost_nothing(dtype, new, dim, profile):
    """softmax1 with every score far below its implicit zero logit: the small outputs keep their precision."""
    b = Batch(new, [6000, 900], seed=56, hkv=1, dim=dim, dtype=dtype, stale=0.0)
    _low_scores(b, LOW_SCORES[profile])
    _chunk_case(b, "softmax1")


@pytest.mark.parametrize("norm", ["sparsemax", "entmax15"])
@pytest.mark.parametrize("kw", [dict(dtype=torch.float32), dict(dim=40), dict(dim=64), dict(dtype=torch.float16, page=5)])
@pytest.mark.parametrize("gain", [0.1, 1.0])
def test_nearly_even_rows(gain, kw, norm):
    """Scores so close that every key is in the support, on every route."""
    _chunk_case(Batch([7, 1, 30], [2471, 720, 735], seed=65, hkv=1, gain=gain, **kw), norm, scale=1e-3)


@pytest.mark.parametrize("norm", ["sparsemax", "entmax15"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_supports_of_very_many_keys(norm, dtype):
    """Even rows over a long context: every probability lies among float16's subnormal numbers."""
    b = Batch([1], [83677], seed=62, group=1, hkv=1, dim=64, page=64, dtype=dtype, stale=0.0)
    b.value_cache = b.value_cache.abs()
    b.d_value = b.value_cache.cuda()
    _chunk_case(b, norm, scale=1e-12)


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim,offset", [(128, 0), (64, 0), (40, 0), (20, 0), (128, 1)])
def test_append(dtype, dim, offset):
    b = Batch([3, 0, 40, 1], [3, 9, 77, 33], dim=dim, dtype=dtype, seed=20, stale=7.0, interleave=dim == 64)
    g = torch.Generator().manual_seed(1)
    total = sum(b.new)
    both = torch.randn(total, 2, b.hkv, dim + 2 * offset, generator=g).to(dtype)[..., offset:offset + dim]
    kc, vc, kw = b.key_cache.clone(), b.value_cache.clone(), b.weights.clone()
    for s, (n, c) in enumerate(zip(b.new, b.lens)):
        rows, t = b.rows[s][c - n:], int(b.cu[s])
        kc[rows], vc[rows], kw[:, rows] = both[t:t + n, 0], both[t:t + n, 1], 0.0
    dev = torch.randn(total, 2, b.hkv, dim + 2 * offset).to(dtype).cuda()[..., offset:offset + dim]
    dev.copy_(both)
    serving.paged_append(dev[:, 0], dev[:, 1], b.d_key, b.d_value, b.d_table, b.d_cu, b.d_seq, b.page,
                         key_weights=b.d_weights)
    assert torch.equal(b.d_key.cpu(), kc) and torch.equal(b.d_value.cpu(), vc) and torch.equal(b.d_weights.cpu(), kw)
    serving.paged_append(dev[:, 0], dev[:, 1], b.d_key, b.d_value, b.d_table, b.d_cu, b.d_seq, b.page)
    assert torch.equal(b.d_weights.cpu(), kw) and serving.device_status() == 0


def test_append_nothing_and_too_much():
    b = Batch([0, 0], [5, 0], seed=21, stale=1.0)
    kc = b.d_key.clone()
    e = torch.zeros(0, b.hkv, b.dim, dtype=b.dtype, device="cuda")
    serving.paged_append(e, e, b.d_key, b.d_value, b.d_table, b.d_cu, b.d_seq, b.page)
    assert torch.equal(b.d_key, kc) and serving.device_status() == 0
    assert b.chunk("softmax1").shape == (0, 8, 128)
    b = Batch([6], [4], seed=22)  # two more tokens than keys: they have no position
    x = torch.randn(6, b.hkv, b.dim).to(b.dtype).cuda()
    serving.paged_append(x, x, b.d_key, b.d_value, b.d_table, b.d_cu, b.d_seq, b.page)
    assert torch.equal(b.d_key[b.rows[0].cuda()], x[2:]) and serving.device_status() == 3


# ---------------------------------------------------------------------------
# evict
# ---------------------------------------------------------------------------
def _evict_expected(b, budget, recent):
    kc, vc, kw = b.key_cache.clone(), b.value_cache.clone(), b.weights.clone()
    kept = np.full((len(b.lens), b.hkv, budget), -1, dtype=np.int32)
    for s, c in enumerate(b.lens):
        for h in range(b.hkv):
            if c <= budget:
                kept[s, h, :c] = np.arange(c)
                continue
            late = min(recent, budget)
            w = b.weights[h, b.rows[s]].double().numpy()[:c - late]
            w = np.where(np.isnan(w), np.inf, w) + 0.0
            nan = np.isnan(b.weights[h, b.rows[s]].numpy()[:c - late])
            order = np.lexsort((np.arange(c - late), -w, ~nan))  # NaN first, then large weights, then low positions
            keep = np.sort(np.concatenate([order[:budget - late], np.arange(c - late, c)]))
            kept[s, h] = keep
            dst, src = b.rows[s][:budget], b.rows[s][torch.from_numpy(keep)]
            kc[dst, h], vc[dst, h], kw[h, dst] = b.key_cache[src, h], b.value_cache[src, h], b.weights[h, src]
    return kept, kc, vc, kw


def _evict_case(b, budget, recent, **kw_args):
    kept, kc, vc, kw = _evict_expected(b, budget, recent)
    lens, got = serving.paged_evict(b.d_key, b.d_value, b.d_weights, b.d_table, b.d_seq, b.page, budget, recent=recent,
                                    **kw_args)
    assert lens.tolist() == [min(c, budget) for c in b.lens]
    np.testing.assert_array_equal(got.cpu().numpy(), kept)
    for actual, want in ((b.d_key, kc), (b.d_value, vc), (b.d_weights, kw)):
        np.testing.assert_array_equal(actual.float().cpu().numpy(), want.float().numpy())
    assert serving.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("budget,recent", [(1, 0), (1, 1), (64, 0), (64, 17), (64, 64), (64, 100), (299, 5), (300, 0),
                                           (1000, 10)])
def test_evict(budget, recent, dtype):
    _evict_case(Batch([1, 1, 1, 0, 1], [300, 64, 65, 0, 7], dtype=dtype, seed=30), budget, recent, max_seqlen_k=300)


@pytest.mark.parametrize("kw", [dict(dim=64, page=16), dict(dim=40), dict(dim=20, page=5), dict(interleave=True), dict(hkv=1)])
def test_evict_layouts(kw):
    _evict_case(Batch([1, 1], [1500, 700], seed=31, **kw), 333, 20)


def test_evict_ties_zeros_infinities_and_nan():
    b = Batch([1, 1, 1], [2100, 2100, 500], seed=32)
    w = torch.randint(0, 3, b.weights.shape, generator=torch.Generator().manual_seed(2)).float()  # many ties
    w[:, b.rows[1]] = 0.0                                     # all equal
    w[0, b.rows[1][5::7]] = -0.0                              # equal to +0
    w[:, b.rows[2][3]], w[:, b.rows[2][400]] = float("inf"), float("nan")
    w[:, b.rows[2][10]] = -1.0
    b.weights = w
    b.d_weights = w.cuda()
    _evict_case(b, 450, 9)


def _evict_around_the_default_shared_memory():
    for keys in (10172, 10173, 10240, 10241):
        _evict_case(Batch([1], [keys], seed=54, hkv=1, dim=64), 300, 7, max_seqlen_k=keys)


def test_evict_around_the_default_shared_memory():
    """The selection's static and dynamic shared memory pass what a launch may have without asking.

    In a process of its own: once a kernel was given more, it keeps it."""
    import multiprocessing

    child = multiprocessing.get_context("spawn").Process(target=_evict_around_the_default_shared_memory)
    child.start()
    child.join(300)
    assert child.exitcode == 0


def test_evict_longer_than_shared_memory_holds():
    """Past 45056 candidates the selection reads the rest of the weights again in every pass."""
    _evict_case(Batch([1], [50000], seed=33, hkv=1, dim=64, page=64), 1200, 33)


def test_evict_then_attend():
    """The kept keys are attended exactly as a cache that only ever held them."""
    b = Batch([2, 3], [200, 90], seed=34)
    lens, kept = serving.paged_evict(b.d_key, b.d_value, b.d_weights, b.d_table, b.d_seq, b.page, 50, recent=8)
    b.key_cache, b.value_cache = b.d_key.cpu(), b.d_value.cpu()
    b.weights, b.d_seq = b.d_weights.cpu(), lens
    b.lens = lens.tolist()
    b.rows = [r[:c] for r, c in zip(b.rows, b.lens)]
    for norm in NORMS:
        b.d_weights = b.weights.cuda()
        _chunk_case(b, norm)


@pytest.mark.parametrize("norm", NORMS)
@pytest.mark.parametrize("new", [[2], [50]])
def test_no_keys_at_all(norm, new):
    b = Batch(new, [0], seed=51)
    for kw in (dict(), dict(max_seqlen_k=0)):
        w = b.weights.cuda()
        assert (b.chunk(norm, key_weights=w, **kw) == 0).all() and torch.equal(w.cpu(), b.weights)
    assert serving.device_status() == 0


@pytest.mark.parametrize("norm", NORMS)
@pytest.mark.parametrize("new", [[1, 2], [60, 70]])
def test_bad_offsets_stay_inside_the_packed_rows(norm, new):
    """Offsets past the packed rows, and rows that belong to no sequence: recorded, and nothing outside is touched."""
    b = Batch(new, [200, 300], seed=52)
    serving.device_status()
    b.d_cu = torch.tensor([-3, new[0], 10 ** 6], dtype=torch.int32, device="cuda")
    b.chunk(norm, key_weights=b.d_weights)
    assert serving.device_status() == 3
    b.d_cu = torch.tensor([0, new[0], new[0]], dtype=torch.int32, device="cuda")
    out, want = b.chunk(norm), b.expected(norm)
    _check(out[:new[0]], want[0][:new[0]], want[1][:new[0]], norm)
    assert serving.device_status() == 0


@pytest.mark.parametrize("norm", NORMS)
@pytest.mark.parametrize("kw", [dict(), dict(dtype=torch.float32)])
@pytest.mark.parametrize("new", [[1, 2], [60, 70], [3] + [0] * 40 + [1]])
def test_decreasing_offsets_are_recorded(new, kw, norm):
    """A sequence whose offsets decrease has no tokens, rows before both are served, and the status tells."""
    b = Batch(new, [200] * len(new), seed=64, **kw)
    want, tol, _, _ = b.expected(norm)
    serving.device_status()
    for end in (new[0] - 1, -5):
        b.d_cu[-1] = end
        out = b.chunk(norm)
        assert serving.device_status() == 3
        _check(out[:new[0] - 1], want[:new[0] - 1], tol[:new[0] - 1], norm) if end >= 0 and new[0] > 1 else None


def test_offsets_past_32_bits():
    """A cache of more than 2^32 bytes and 2^31 elements, its pages in use at the far end: the same bits as in a small one."""
    small = Batch([70, 1, 3], [400, 600, 131], seed=50, hkv=8, group=2, interleave=True, stale=0.0)
    slots = small.key_cache.shape[0]
    far = (2 ** 31 // (2 * 8 * 128) // 32 + 1) * 32  # the first page whose element offsets pass 2^31
    both = torch.empty(far + slots, 2, 8, 128, dtype=small.dtype, device="cuda")
    both[far:, 0], both[far:, 1] = small.d_key, small.d_value
    weights = torch.zeros(8, far + slots, device="cuda")
    weights[:, far:] = small.d_weights
    table = (small.d_table + far // 32).to(torch.int32)
    new = torch.randn(74, 2, 8, 128, device="cuda").to(small.dtype)

    def run(kc, vc, w, table):
        serving.paged_append(new[:, 0], new[:, 1], kc, vc, table, small.d_cu, small.d_seq, 32, key_weights=w)
        outs = [serving.paged_chunk_attention(small.d_query, kc, vc, table, small.d_cu, small.d_seq, 32, norm, key_weights=w,
                                              max_seqlen_q=n) for norm in NORMS for n in (70, 1)]
        outs += serving.paged_evict(kc, vc, w, table, small.d_seq, 32, 100, recent=5)
        return outs + [kc[-slots:], vc[-slots:], w[:, -slots:]]

    for a, b in zip(run(small.d_key, small.d_value, small.d_weights, small.d_table), run(both[:, 0], both[:, 1], weights, table)):
        assert torch.equal(a, b)
    assert serving.device_status() == 0


@pytest.mark.parametrize("norm", NORMS)
@pytest.mark.parametrize("new", [[1, 1, 1], [40, 1, 90]])
def test_pages_rewritten_back_to_back(norm, new):
    """Each call reads what the one before it wrote into the same pages, launched while that one still runs."""
    rows = torch.randn(12, sum(new), 2, 2, 128, generator=torch.Generator().manual_seed(3)).bfloat16().cuda()

    def run(pause):
        b = Batch(new, [300, 700, 260], seed=63, gain=2.0)
        outs = []
        for x in rows:
            serving.paged_append(x[:, 0], x[:, 1], b.d_key, b.d_value, b.d_table, b.d_cu, b.d_seq, b.page,
                                 key_weights=b.d_weights)
            pause()
            outs.append(b.chunk(norm, key_weights=b.d_weights))
            pause()
        for budget in range(240, 100, -20):
            b.d_seq, _ = serving.paged_evict(b.d_key, b.d_value, b.d_weights, b.d_table, b.d_seq, b.page, budget, recent=95)
            pause()
            outs.append(b.chunk(norm, key_weights=b.d_weights))
            pause()
        return outs + [b.d_weights]

    for got, want in zip(run(lambda: None), run(torch.cuda.synchronize)):
        assert torch.equal(got, want)
    assert serving.device_status() == 0


# ---------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------
def test_gradients_are_refused():
    b = Batch([2], [20], seed=40)
    b.d_query.requires_grad_(True)
    with pytest.raises(ValueError, match="inference only"):
        b.chunk("softmax1")
    with torch.no_grad():
        assert torch.isfinite(b.chunk("softmax1")).all()


def test_64_bit_integers_past_32_bits_are_recorded():
    """Lengths, offsets and page ids that a cut to 32 bits would turn into valid ones."""
    b = Batch([3, 1], [60, 40], seed=61)
    out = b.chunk("softmax1")
    b.d_table, b.d_cu, b.d_seq = b.d_table.long(), b.d_cu.long(), b.d_seq.long()
    assert torch.equal(b.chunk("softmax1"), out) and serving.device_status() == 0
    for field, at, status in (("d_table", (0, 0), 1), ("d_seq", 0, 3), ("d_cu", 2, 3)):
        t = getattr(b, field)
        for by in (2 ** 32, -2 ** 32):
            t[at] += by
            b.chunk("softmax1")
            assert serving.device_status() == status, field
            t[at] -= by
    new = torch.randn(4, b.hkv, b.dim, device="cuda").to(b.dtype)
    key = b.d_key.clone()
    b.d_table[:, :2] += 2 ** 32
    serving.paged_append(new, new, b.d_key, b.d_value, b.d_table, b.d_cu, b.d_seq, b.page)
    assert torch.equal(b.d_key.nan_to_num(), key.nan_to_num()) and serving.device_status() == 1
    b.d_table[:, :2] -= 2 ** 32
    lens, _ = serving.paged_evict(b.d_key, b.d_value, b.d_weights, b.d_table, b.d_seq + 2 ** 32, b.page, 50)
    assert lens.tolist() == [50, 50] and serving.device_status() == 3


@pytest.mark.parametrize("norm", NORMS)
def test_written_tensors_raise_their_versions(norm):
    """Autograd has to notice that a cache it saved was written."""
    b = Batch([3, 1], [60, 40], seed=58)
    new = torch.randn(4, b.hkv, b.dim, device="cuda").to(b.dtype)

    def versions():
        return [t._version for t in (b.d_key, b.d_value, b.d_weights)]

    was = versions()
    serving.paged_append(new, new, b.d_key, b.d_value, b.d_table, b.d_cu, b.d_seq, b.page, key_weights=b.d_weights)
    now = versions()
    assert all(a > w for a, w in zip(now, was))
    b.chunk(norm, key_weights=b.d_weights)
    assert versions()[:2] == now[:2] and versions()[2] > now[2]
    was = versions()
    serving.paged_evict(b.d_key, b.d_value, b.d_weights, b.d_table, b.d_seq, b.page, 20)
    assert all(a > w for a, w in zip(versions(), was))

    factor = torch.ones((), device="cuda", dtype=b.dtype, requires_grad=True)
    y = b.d_key * factor  # saves the cache
    with torch.no_grad():
        serving.paged_append(new, new, b.d_key, b.d_value, b.d_table, b.d_cu, b.d_seq, b.page)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_inference_mode():
    """Tensors without a version counter."""
    with torch.inference_mode():
        b = Batch([3, 1], [60, 40], seed=59)
        new = torch.randn(4, b.hkv, b.dim, device="cuda").to(b.dtype)
        serving.paged_append(new, new, b.d_key, b.d_value, b.d_table, b.d_cu, b.d_seq, b.page, key_weights=b.d_weights)
        b.key_cache, b.value_cache, b.weights = b.d_key.cpu(), b.d_value.cpu(), b.d_weights.cpu()
        _chunk_case(b, "softmax1")
        serving.paged_evict(b.d_key, b.d_value, b.d_weights, b.d_table, b.d_seq, b.page, 20)


def test_dispatch_modes_and_the_profiler_see_the_calls():
    from torch.utils._python_dispatch import TorchDispatchMode

    b = Batch([3, 1], [60, 40], seed=60)
    new = torch.randn(4, b.hkv, b.dim, device="cuda").to(b.dtype)

    def step():
        serving.paged_append(new, new, b.d_key, b.d_value, b.d_table, b.d_cu, b.d_seq, b.page, key_weights=b.d_weights)
        b.chunk("softmax1", key_weights=b.d_weights)
        serving.paged_evict(b.d_key, b.d_value, b.d_weights, b.d_table, b.d_seq, b.page, 20)

    names = ["hfan::paged_append", "hfan::paged_chunk_fwd", "hfan::paged_evict"]
    seen = []

    class Log(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(func.name())
            return func(*args, **(kwargs or {}))

    with Log():
        step()
    assert [n for n in seen if n.startswith("hfan::")] == names
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]) as prof:
        step()
    assert set(names) <= {e.name for e in prof.events()}


def test_tensors_elsewhere_are_refused():
    b = Batch([2], [20], seed=41)
    with pytest.raises(ValueError, match="requires CUDA"):
        serving.paged_chunk_attention(b.query, b.key_cache, b.value_cache, b.table, b.cu, b.seq, b.page)
    with pytest.raises(ValueError, match="one device"):
        serving.paged_chunk_attention(b.d_query, b.d_key, b.d_value, b.table, b.d_cu, b.d_seq, b.page)


# ---------------------------------------------------------------------------
# the cache and the example, as a user runs them
# ---------------------------------------------------------------------------
def _example():
    import importlib.util
    import os

    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "serve_paged.py")
    spec = importlib.util.spec_from_file_location("serve_paged", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("norm", NORMS)
def test_serving_a_model_matches_its_full_forward(norm):
    """Prompt pieces and single tokens through the pages give the logits of one pass over the whole text.

    Both run in bfloat16 through the same layers; only the attention's own rounding differs, a few units of 2^-8
    of a hidden state whose logits have unit scale.
    """
    import hf_attention_normalizers_b200 as H

    ex = _example()
    model = ex.small_model(layers=2)
    texts = [torch.randint(0, 1024, (n,), generator=torch.Generator().manual_seed(n)).tolist() for n in (150, 37, 1)]
    plan = [[64, 37, 0], [64, 0, 1], [21, 0, 0], [1, 0, 0]]
    c = model.config
    cache = serving.PagedServingCache(2, 3, 12, 32, c.num_key_value_heads, c.head_dim)
    got = [[], [], []]
    with torch.no_grad():
        at = [0, 0, 0]
        for counts in plan:
            step = cache.step(counts)
            ids = torch.tensor([t for s, p, n in zip(texts, at, counts) for t in s[p:p + n]], device="cuda")
            pos = torch.tensor([p + i for p, n in zip(at, counts) for i in range(n)], device="cuda")
            logits = ex.forward_step(model, cache, step, ids, pos, norm).float()
            for b, part in enumerate(logits.split(counts)):
                got[b].append(part)
                at[b] += counts[b]
        H.set_softmax_attention_backend(model, base_backend="sdpa", softmax_fn=norm)
        for text, parts in zip(texts, got):
            want = model(torch.tensor([text], device="cuda")).logits[0].float()
            have = torch.cat(parts)
            assert have.shape == want.shape
            assert (have - want).norm() <= 2.0 ** -5 * want.norm()


@pytest.mark.parametrize("norm", NORMS)
def test_serving_under_a_budget_frees_pages(norm):
    ex = _example()
    model = ex.small_model(layers=2)
    prompts = [list(range(300)), list(range(40)), [5]]
    free = ex.generate(model, prompts, 6, norm, piece=64)
    # a budget that nothing exceeds changes nothing; a small one runs in the memory of the budget alone
    assert ex.generate(model, prompts, 6, norm, piece=64, budget=400) == free
    cut = ex.generate(model, prompts, 6, norm, piece=64, budget=96, recent=16)
    assert [len(o) for o in cut] == [6, 6, 6] and serving.device_status() == 0


def test_cache_bookkeeping():
    cache = serving.PagedServingCache(1, 2, 6, 16, 1, 64, track_weights=True)
    step = cache.step([40, 16])
    assert cache.lengths == [40, 16] and step.max_seqlen_q == 40 and step.max_seqlen_k == 40
    assert step.cu_seqlens.tolist() == [0, 40, 56] and step.lengths.tolist() == [40, 16]
    with pytest.raises(ValueError, match="no room"):
        cache.step([40, 16])
    with pytest.raises(ValueError, match="one count per sequence"):
        cache.step([1])
    cache.evict(20, 4)
    assert cache.lengths == [20, 16]
    step = cache.step([12, 33])  # 32 and 49 tokens: six pages again
    assert cache.lengths == [32, 49] and len(set(step.block_table[0, :2].tolist() + step.block_table[1, :4].tolist())) == 6
    with pytest.raises(ValueError, match="track_weights"):
        serving.PagedServingCache(1, 1, 2, 16, 1, 64).evict(4)
