"""Kernels behind sampling several continuations of one prompt, against plain forms in 64 bits: shared-prefix
attention, page copies, pool compaction, verification of drafted tokens."""
import math
import random

import pytest
import torch

from mod_b200.ops import reference as R

pytestmark = pytest.mark.gpu

PAGE = 16


@pytest.fixture(scope="module")
def N(cuda):
    from mod_b200.ops import native

    native._C()
    return native


@pytest.fixture(autouse=True)
def no_status(cuda):
    from mod_b200.ops import check_status

    yield
    torch.cuda.synchronize()
    check_status()


@pytest.fixture(scope="module")
def cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda:0")


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------ attention
class Batch:
    """Groups as (prefix tokens, [(own tokens, query tokens), ...]); an own length of None is a padded row.  Token
    slots that no sequence holds are NaN in both caches."""

    def __init__(self, groups, Hq, Hkv, D, seed=0, q_scale=2.0, base=0, spare=3):
        r = random.Random(seed)
        g = torch.Generator(device="cuda").manual_seed(seed)
        rows, self.ctx, self.nq, self.offs, self.shared = [], [], [], [0], []
        total = sum(p // PAGE + sum(-(-(p % PAGE + (o or 0)) // PAGE) for o, _ in seqs) for p, seqs in groups) + spare
        ids = list(range(base, base + total))
        r.shuffle(ids)
        self.k = torch.full((base + total, Hkv, PAGE, D), math.nan, dtype=torch.bfloat16, device="cuda")
        self.v = torch.full((base + total, Hkv, D, PAGE), math.nan, dtype=torch.bfloat16, device="cuda")

        def fill(page, tokens):
            self.k[page, :, :tokens] = torch.randn(Hkv, tokens, D, device="cuda", generator=g).bfloat16()
            self.v[page, :, :, :tokens] = torch.randn(Hkv, D, tokens, device="cuda", generator=g).bfloat16()

        for p, seqs in groups:
            common = [ids.pop() for _ in range(p // PAGE)]
            for c in common:
                fill(c, PAGE)
            for o, n in seqs:
                left = 0 if o is None else p % PAGE + o
                row = list(common)
                while left > 0:
                    row.append(ids.pop())
                    fill(row[-1], min(PAGE, left))
                    left -= PAGE
                rows.append(row)
                self.ctx.append(0 if o is None else p + o)
                self.nq.append(n)
            self.offs.append(len(rows))
            self.shared.append(p)
        width = max(1, max(len(x) for x in rows)) + 1
        self.tables = ints([x + [0] * (width - len(x)) for x in rows])
        self.cu = [0]
        for n in self.nq:
            self.cu.append(self.cu[-1] + n)
        self.q = (torch.randn(self.cu[-1], Hq, D, device="cuda", generator=g) * q_scale).bfloat16()

    def plan(self, N, share=True, cu=True):
        T, Hq, D = self.q.shape
        shared = ints(self.shared if share else [0] * len(self.shared))
        return N.attn_shared_plan(self.tables, ints(self.ctx), ints(self.offs), shared, T, Hq, self.k.shape[1], D,
                                  cu_q=ints(self.cu) if cu else None)

    def check(self, out, scale=None):
        """Every output against 64 bits.  Rounding the weights to bf16 costs at most 2^-9 of sum(p |v|), rounding the
        output 2^-9 of it again; 2^-11 more covers the 32-bit exponentials and sums of scores up to a few hundred."""
        T, Hq, D = self.q.shape
        rep = Hq // self.k.shape[1]
        scale = 1 / math.sqrt(D) if scale is None else scale
        assert not torch.isnan(out).any()
        for b, c in enumerate(self.ctx):
            t0, t1 = self.cu[b], self.cu[b + 1]
            if c == 0:
                assert (out[t0:t1] == 0).all()
                continue
            k = R.gather_kv(self.k, self.tables[b], c).double().repeat_interleave(rep, 1)
            v = R.gather_v(self.v, self.tables[b], c).double().repeat_interleave(rep, 1)
            s = torch.einsum("qhd,nhd->hqn", self.q[t0:t1].double(), k) * scale
            seen = torch.arange(c, device="cuda")[None, :] <= c - (t1 - t0) + torch.arange(t1 - t0, device="cuda")[:, None]
            p = torch.softmax(s.masked_fill(~seen[None], -math.inf), -1)
            o = torch.einsum("hqn,nhd->qhd", p, v)
            bound = torch.einsum("hqn,nhd->qhd", p, v.abs()) * (2 ** -8 + 2 ** -11) + 1e-6
            err = (out[t0:t1].double() - o).abs()
            assert (err <= bound).all(), (b, c, float((err / bound).max()))


def seqs(*own, n=1):
    return [(o, n) for o in own]


SHAPES = {
    "one key": [(0, seqs(1))],
    "short": [(5, seqs(1, 2, 11, 12))],
    "no prefix": [(0, seqs(1, 15, 16, 17, 127, 128, 129, 300))],
    "one page": [(16, seqs(1, 16, 40))],
    "tile edges": [(127, seqs(1, 3)), (128, seqs(2, 129)), (129, seqs(128, 1)), (143, seqs(1)), (144, seqs(130, 7, 8))],
    "padded rows": [(33, seqs(4, 9)), (0, seqs(None)), (200, seqs(5)), (0, seqs(None)), (0, seqs(None))],
    "all padded": [(0, seqs(None)), (0, seqs(None))],
    "long": [(5003, seqs(1, 700, 33))],
    "many": [(1000, seqs(*range(1, 70)))],
    "many groups": [(17 * i, seqs(*range(1 + i % 5, 9))) for i in range(20)],
    "drafts": [(300, [(5, 5), (9, 3), (40, 1), (4, 4)]), (64, [(130, 2), (8, 8)])],
    "prefill": [(32, [(150, 150), (300, 290)]), (0, [(200, 200)])],
}


@pytest.mark.parametrize("heads", [(8, 2, 128), (16, 16, 128), (6, 2, 128), (32, 4, 128), (40, 2, 128), (4, 1, 64),
                                   (16, 2, 256), (3, 3, 256)], ids=str)
@pytest.mark.parametrize("shape", SHAPES)
def test_attn_shared(N, shape, heads):
    b = Batch(SHAPES[shape], *heads, seed=len(shape))
    b.check(N.attn_shared(b.q, b.k, b.v, b.tables, b.plan(N)))


def test_attn_shared_many_rows(N):
    # more rows a group than one tile holds, several KV heads, two prompts
    b = Batch([(2100, seqs(*[1 + i % 37 for i in range(100)])), (640, seqs(*[3] * 28))], 32, 4, 128, seed=3)
    b.check(N.attn_shared(b.q, b.k, b.v, b.tables, b.plan(N, cu=False)))


@pytest.mark.parametrize("q_scale", [0.0, 30.0], ids=["equal", "peaked"])
def test_attn_shared_scores(N, q_scale):
    b = Batch([(700, seqs(5, 200, 31))], 16, 4, 128, seed=5, q_scale=q_scale)
    b.check(N.attn_shared(b.q, b.k, b.v, b.tables, b.plan(N)))


def test_attn_shared_rising_scores(N):
    # every tile's scores are far above those of the tile before it, so that the running maximum keeps moving
    b = Batch([(1024, seqs(40, 200))], 8, 2, 128, seed=6)
    b.q.fill_(1.0)
    for row, c in zip(b.tables.tolist(), b.ctx):
        for j in range(-(-c // PAGE)):
            b.k[row[j], :, :min(PAGE, c - j * PAGE)] = j / 4
    b.check(N.attn_shared(b.q, b.k, b.v, b.tables, b.plan(N)))


def test_attn_shared_scale_and_out(N):
    b = Batch([(90, seqs(3, 50))], 8, 2, 128, seed=7)
    out = torch.full_like(b.q, math.nan)
    assert N.attn_shared(b.q, b.k, b.v, b.tables, b.plan(N), out=out, scale=0.3) is out
    b.check(out, scale=0.3)


def test_attn_shared_is_what_the_tables_say(N):
    # a promise to share changes what is read, not the result
    b = Batch([(500, seqs(20, 7, 90))], 8, 2, 128, seed=8)
    b.check(N.attn_shared(b.q, b.k, b.v, b.tables, b.plan(N, share=False)))


def test_attn_shared_prefix_longer_than_a_context(N):
    # shared_lens past a sequence's first query token only promises equal tables
    b = Batch([(0, [(40, 1)]), (0, [(64, 30)])], 8, 2, 128, seed=9)
    b.shared = [40, 64]
    b.check(N.attn_shared(b.q, b.k, b.v, b.tables, b.plan(N)))


def test_attn_shared_fewer_tokens_than_queries(N):
    # query tokens that lie before the context's first token see nothing
    b = Batch([(0, [(8, 8), (40, 40), (5, 1)])], 8, 2, 128, seed=13)
    b.ctx = [3, 30, 5]
    out = N.attn_shared(b.q, b.k, b.v, b.tables, b.plan(N))
    assert (out[:5] == 0).all() and (out[8:18] == 0).all()
    for t0, t1, c, row in ((5, 8, 3, 0), (18, 48, 30, 1), (48, 49, 5, 2)):
        part = Batch.__new__(Batch)
        part.q, part.k, part.v, part.tables = b.q[t0:t1], b.k, b.v, b.tables[row:row + 1]
        part.ctx, part.cu = [c], [0, t1 - t0]
        part.check(out[t0:t1])


def test_attn_shared_lengths_that_do_not_fit_are_reported(N):
    from mod_b200.ops import check_status

    b = Batch([(64, seqs(5, 6, 7, 8))], 8, 2, 128, seed=14)
    T, Hq, D = b.q.shape
    for cu, offs in (([0, 4, 0, 4, 0], [0, 4]), ([0, 1, 2, 3, 4], [0, 4, 0, 4, 0, 4])):
        p = N.attn_shared_plan(b.tables, ints(b.ctx), ints(offs), ints([64] * (len(offs) - 1)), T, Hq, 2, D, cu_q=ints(cu))
        out = N.attn_shared(b.q, b.k, b.v, b.tables, p)
        with pytest.raises(RuntimeError, match="out of bounds"):
            check_status()
        assert (out == 0).all()
    # a page that there is none of counts as masked
    b.tables[0, 4] = 10 ** 6
    N.attn_shared(b.q, b.k, b.v, b.tables, b.plan(N))
    with pytest.raises(RuntimeError, match="out of bounds"):
        check_status()


def test_attn_shared_repeats_bit_for_bit(N):
    b = Batch([(3000, seqs(*range(1, 40)))], 16, 4, 128, seed=10)
    p = b.plan(N)
    first = N.attn_shared(b.q, b.k, b.v, b.tables, p)
    for _ in range(5):
        assert torch.equal(first, N.attn_shared(b.q, b.k, b.v, b.tables, p))


def test_attn_shared_far_pages(N):
    # page offsets past 2^32 bytes and 2^31 elements
    b = Batch([(300, seqs(20, 7))], 8, 2, 128, seed=11, base=1_060_000)
    assert b.k.numel() > 2 ** 32
    b.check(N.attn_shared(b.q, b.k, b.v, b.tables, b.plan(N)))


def test_attn_shared_streams_and_graph(N):
    b = Batch([(200, seqs(20, 7, 55))], 8, 2, 128, seed=12)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        outs = [N.attn_shared(b.q, b.k, b.v, b.tables, b.plan(N)) for _ in range(3)]
    torch.cuda.current_stream().wait_stream(s)
    for o in outs:
        b.check(o)
    # captured with one context, replayed with others: the plan is made from the device's lengths
    ctx, tables = ints(b.ctx), b.tables
    offs, shared = ints(b.offs), ints(b.shared)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        p = N.attn_shared_plan(tables, ctx, offs, shared, 3, 8, 2, 128)
        out = N.attn_shared(b.q, b.k, b.v, tables, p)
    for less in (0, 3, 6):
        b.ctx = [220 - less, 207 - less, 255 - less]
        ctx.copy_(ints(b.ctx))
        graph.replay()
        b.check(out)


def test_attn_shared_refuses(N):
    b = Batch([(20, seqs(3, 5))], 8, 2, 128)
    p = b.plan(N)
    for bad in (b.q[:1], b.q[:, :4], b.q.float()):
        with pytest.raises((ValueError, RuntimeError)):
            N.attn_shared(bad.contiguous(), b.k, b.v, b.tables, p)
    with pytest.raises((ValueError, RuntimeError)):
        N.attn_shared(b.q, b.k.transpose(2, 3), b.v, b.tables, p)
    with pytest.raises((ValueError, RuntimeError)):
        N.attn_shared(b.q, b.k, b.v, b.tables[:, :1].contiguous(), p)
    with pytest.raises((ValueError, RuntimeError)):
        N.attn_shared(b.q.transpose(0, 1).contiguous().transpose(0, 1), b.k, b.v, b.tables, p)
    with pytest.raises((ValueError, RuntimeError)):
        N.attn_shared_plan(b.tables, ints(b.ctx).long(), ints(b.offs), ints(b.shared), 2, 8, 2, 128)
    with pytest.raises((ValueError, RuntimeError)):
        N.attn_shared_plan(b.tables, ints(b.ctx), ints(b.offs), ints(b.shared), 3, 8, 2, 128)
    with pytest.raises((ValueError, RuntimeError)):
        N.attn_shared_plan(b.tables, ints(b.ctx), ints(b.offs), ints(b.shared), 2, 8, 2, 96)
    with pytest.raises((ValueError, RuntimeError)):
        N.attn_shared_plan(b.tables, ints(b.ctx), ints(b.offs[:1]), ints(b.shared), 2, 8, 2, 128)


# ------------------------------------------------------------------ pages
def caches(layers, pages, heads, D, dtype=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(layers)
    k = [torch.randn(pages, heads, PAGE, D, device="cuda", generator=g).to(dtype) for _ in range(layers)]
    v = [torch.randn(pages, heads, D, PAGE, device="cuda", generator=g).to(dtype) for _ in range(layers)]
    return k, v


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("layers,heads,D", [(1, 1, 8), (3, 2, 128), (70, 1, 64), (2, 8, 256), (2, 3, 40)])
def test_copy_pages(N, layers, heads, D, dtype):
    k, v = caches(layers, 23, heads, D, dtype)
    k[0][4].fill_(math.nan)
    want_k, want_v = [x.clone() for x in k], [x.clone() for x in v]
    src, dst = ints([4, 4, 22, -1, 7, 0]), ints([1, 2, 0 + 3, 5, -1, 21])
    R.kv_copy_pages(want_k, want_v, src, dst)
    N.kv_copy_pages(k, v, src, dst)
    for a, b in zip(k + v, want_k + want_v):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_copy_pages_none_and_far(N):
    k, v = caches(1, 4, 2, 128)
    before = [x.clone() for x in k + v]
    N.kv_copy_pages(k, v, ints([]), ints([]))
    assert all(torch.equal(a, b) for a, b in zip(before, k + v))
    pages = 140_000  # 4.6 GB a cache: offsets past 2^32 bytes and 2^31 elements
    k, v = ([torch.zeros(pages, 8, *s, dtype=torch.bfloat16, device="cuda")] for s in ((PAGE, 128), (128, PAGE)))
    k[0][pages - 1], v[0][pages - 1], k[0][5], v[0][5] = 1.0, 2.0, 3.0, 4.0
    N.kv_copy_pages(k, v, ints([pages - 1, 5]), ints([0, pages - 2]))
    assert (k[0][0] == 1).all() and (v[0][0] == 2).all()
    assert (k[0][pages - 2] == 3).all() and (v[0][pages - 2] == 4).all()
    assert (k[0][1] == 0).all() and (k[0][pages - 3] == 0).all()


def test_copy_pages_out_of_range_is_reported(N):
    from mod_b200.ops import check_status

    k, v = caches(2, 4, 2, 128)
    before = [x.clone() for x in k + v]
    N.kv_copy_pages(k, v, ints([0, 9]), ints([4, 1]))
    with pytest.raises(RuntimeError, match="out of bounds"):
        check_status()
    assert all(torch.equal(a, b) for a, b in zip(before, k + v))


def test_copy_pages_refuses(N):
    k, v = caches(2, 4, 2, 128)
    one = ints([1])
    for args in ((k, v[:1], one, one), ([], [], one, one), (k, v, one, ints([1, 2])), (k, v, one.long(), one),
                 (k, v, one.cpu(), one), ([k[0], k[1][:2]], v, one, one), ([k[0], k[1].float()], v, one, one),
                 ([k[0], k[1].transpose(2, 3)], v, one, one)):
        with pytest.raises(RuntimeError):
            N.kv_copy_pages(*args)


def pool(pages, rows, live, moves, seed):
    """Tables of `rows` rows over exactly `live` pages, `moves` of them at or past `live`; some shared among rows."""
    r = random.Random(seed)
    used = r.sample(range(live), live - moves) + r.sample(range(live, pages), moves)
    r.shuffle(used)
    tables = [[] for _ in range(rows)]
    for p in used:
        tables[r.randrange(rows)].append(p)
    for t in tables[1:]:
        t[:0] = tables[0][:r.randint(0, 3)]
    lens = [max(0, PAGE * len(t) - r.randint(0, PAGE - 1)) for t in tables]
    width = max(len(t) for t in tables) + 2
    # what lies past a row's length is no reference
    return ints([t + [r.randrange(pages) for _ in range(width - len(t))] for t in tables]), ints(lens)


@pytest.mark.parametrize("pages,rows,live,moves", [(1, 1, 1, 0), (2, 1, 1, 1), (16, 3, 0, 0), (16, 4, 16, 0), (40, 5, 20, 20),
                                                   (1000, 7, 500, 250), (1025, 90, 700, 325), (5000, 300, 2500, 2400),
                                                   (70001, 40, 30000, 7)])
def test_compact(N, pages, rows, live, moves):
    heads, D = (1, 8) if pages > 2000 else (2, 64)
    k, v = caches(3, pages, heads, D)
    tables, lens = pool(pages, rows, live, moves, seed=pages)
    old_k, old_v = [x.clone() for x in k], [x.clone() for x in v]
    want_k, want_v = [x.clone() for x in k], [x.clone() for x in v]
    want = R.kv_compact(want_k, want_v, tables, lens)
    keep = tables.clone()
    got = N.kv_compact(k, v, tables, lens)
    assert torch.equal(tables, keep)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    assert int(got[2]) == live
    for a, b in zip(k + v, want_k + want_v):
        assert torch.equal(a, b)
    # what every row holds is what it held
    for r, n in enumerate(lens.tolist()):
        m = -(-n // PAGE)
        for new, old in zip(k + v, old_k + old_v):
            assert torch.equal(new[got[0][r, :m].long()], old[tables[r, :m].long()])
    # once compact, nothing moves; in place
    again = N.kv_compact(k, v, got[0], lens, out=got[0])
    assert again[0] is got[0] and torch.equal(got[0], want[0])
    assert (again[1][:live] == torch.arange(live, device="cuda", dtype=torch.int32)).all()


def test_compact_no_rows_and_bad_pages(N):
    from mod_b200.ops import check_status

    k, v = caches(1, 8, 1, 64)
    _, remap, live = N.kv_compact(k, v, torch.zeros(0, 4, dtype=torch.int32, device="cuda"), ints([]))
    assert int(live) == 0 and (remap == -1).all()
    before = [x.clone() for x in k + v]
    tables, _, live = N.kv_compact(k, v, ints([[0, 8, -3, 1]]), ints([64]))
    with pytest.raises(RuntimeError, match="out of bounds"):
        check_status()
    assert int(live) == 2 and tables.tolist() == [[0, 0, 0, 1]]
    assert all(torch.equal(a, b) for a, b in zip(before, k + v))


def test_compact_refuses(N):
    k, v = caches(2, 8, 1, 64)
    t, n = ints([[0, 1]]), ints([20])
    for args in ((k, v, t.long(), n), (k, v, t, n.long()), (k, v, t, ints([1, 2])), (k, v[:1], t, n), (k, v, t[0], n)):
        with pytest.raises(RuntimeError):
            N.kv_compact(*args)


# ------------------------------------------------------------------ verification
class Drafts:
    def __init__(self, counts, V, heat, seed=0, dtype=torch.float32, q_dtype=None, K=None, spread=2.0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.B, self.V = len(counts), V
        self.K = max(counts) if K is None else K
        self.offs = [0]
        for n in counts:
            self.offs.append(self.offs[-1] + n + 1)
        T = self.offs[-1]
        x = torch.randn(T, V, device="cuda", generator=g) * spread
        likely = torch.randint(0, V, (T,), device="cuda", generator=g)
        x[torch.arange(T), likely] = math.log(V) + spread
        self.logits = x.to(dtype)
        self.cu = ints(self.offs)
        at = torch.tensor([[min(o + j, T - 1) for j in range(self.K)] for o in self.offs[:-1]], dtype=torch.long,
                          device="cuda").view(self.B, self.K)
        some = torch.randint(0, V, (self.B, self.K), device="cuda", generator=g)
        self.drafts = torch.where(torch.rand(self.B, self.K, device="cuda", generator=g) < 0.8, likely[at], some)
        self.uniforms = torch.rand(self.B, self.K, device="cuda", generator=g)
        self.noise = torch.empty(self.B, V, device="cuda").exponential_(generator=g).clamp_(min=1e-20)
        self.heat = torch.tensor(heat * self.B if len(heat) == 1 else heat, device="cuda")
        self.probs = None
        if q_dtype is not None and self.K:
            q = torch.softmax(x[at.reshape(-1)] + torch.randn(self.B * self.K, V, device="cuda", generator=g) * 0.5, -1)
            self.probs = q.view(self.B, self.K, V).to(q_dtype)

    def run(self, N):
        return N.verify_sampled(self.logits, self.cu, self.drafts, self.uniforms, self.noise, self.heat, self.probs)

    def check(self, got):
        """Whole numbers as 64 bits give them (the seeds leave no near ties), probabilities to 2^-18: an exponent of up
        to 40 loses 2^-24 of itself in 32 bits, about 2^-19, the sum and the quotient a few 2^-24 more."""
        for b in range(self.B):
            n, a, t = self.offs[b + 1] - self.offs[b] - 1, 0, float(self.heat[b])
            said = []
            while True:
                x = self.logits[self.offs[b] + a].double()
                p = torch.softmax(x / self.heat[b].double(), 0) if t > 0 else \
                    torch.zeros_like(x).index_fill_(0, x.argmax(), 1.0)
                rest = p
                if a < n:
                    d = int(self.drafts[b, a])
                    q = torch.zeros_like(p).index_fill_(0, torch.tensor(d, device="cuda"), 1.0) if self.probs is None \
                        else self.probs[b, a].double()
                    if float(self.uniforms[b, a].double() * q[d]) < float(p[d]):
                        said.append(float(p[d]))
                        a += 1
                        continue
                    rest = (p - q).clamp(min=0)
                    rest = rest if float(rest.sum()) > 0 else p
                break
            v = int((rest / self.noise[b].double()).argmax())
            said.append(float(p[v]))
            assert int(got[0][b]) == a and int(got[1][b]) == v, (b, n, int(got[0][b]), a, int(got[1][b]), v)
            want = torch.tensor(said + [0.0] * (self.K + 1 - len(said)), dtype=torch.float64)
            err = (got[2][b].double().cpu() - want).abs()
            assert (err <= want * 2 ** -18).all(), (b, err, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("q_dtype", [None, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [1, 2, 31, 512, 1000, 151553])
def test_verify(N, V, q_dtype, dtype):
    x = Drafts([0, 1, 4, 3, 0, 2, 4, 5], V, [0.0, 1.0, 0.7, 1.3, 1.0, 0.0, 0.5, 2.0], seed=V, dtype=dtype, q_dtype=q_dtype)
    x.check(x.run(N))


@pytest.mark.parametrize("counts", [[0], [1], [17], [0, 0, 0], [8] * 40, [i % 5 for i in range(130)]], ids=str)
def test_verify_batches(N, counts):
    x = Drafts(counts, 3001, [0.9], seed=len(counts), dtype=torch.bfloat16)
    x.check(x.run(N))


def test_verify_no_sequences(N):
    x = Drafts([0], 64, [1.0], K=2)
    got = N.verify_sampled(x.logits[:0], x.cu[:1], x.drafts[:0], x.uniforms[:0], x.noise[:0], x.heat[:0])
    assert [tuple(t.shape) for t in got] == [(0,), (0,), (0, 3)]


def test_verify_unused_draft_columns(N):
    x = Drafts([1, 0, 2], 700, [1.0], seed=4, K=6)
    x.drafts[0, 1:] = -5
    x.drafts[1, :] = 10 ** 12
    x.uniforms[2, 2:] = math.nan
    x.check(x.run(N))


def test_verify_accept_all_and_none(N):
    x = Drafts([3, 3], 500, [1.0], seed=5)
    x.uniforms.zero_()
    got = x.run(N)
    assert got[0].tolist() == [3, 3]
    x.check(got)
    x.uniforms.fill_(1 - 2 ** -24)
    x.drafts = torch.full_like(x.drafts, 7)
    got = x.run(N)
    assert got[0].tolist() == [0, 0] and 7 not in got[1].tolist()
    x.check(got)


def test_verify_draft_equals_target(N):
    # q = p: every draft passes whatever its uniform number; refused by an out-of-range id, the rest is empty and p is used
    x = Drafts([2, 2], 300, [1.0], seed=6, q_dtype=torch.float32)
    for b in range(2):
        x.probs[b] = torch.softmax(x.logits[x.offs[b]:x.offs[b] + 2].double(), -1).float() * 0.999
    x.uniforms.fill_(0.999)
    assert x.run(N)[0].tolist() == [2, 2]
    x.probs = (x.probs / 0.999).clamp(min=0) + 1e-3
    x.drafts[0, 0], x.drafts[1, 0] = 300, -1
    acc, tok, _ = x.run(N)
    assert acc.tolist() == [0, 0]
    for b in range(2):
        p = torch.softmax(x.logits[x.offs[b]].double(), 0)
        assert int(tok[b]) == int((p / x.noise[b]).argmax())


def test_verify_greedy_ties_and_masks(N):
    V = 5000
    x = Drafts([2, 1, 1, 1, 0, 2], V, [0.0, 1.0, 1.0, 1.0, 0.0, 1.0], seed=7)
    low, inf = torch.finfo(torch.float32).min, math.inf
    x.logits[0].fill_(low)
    x.logits[0, [4321, 77, 78]] = 3.0               # the lowest of equals wins
    x.logits[1].fill_(-inf)
    x.logits[1, 4999] = -7.0
    x.drafts[0, :2] = torch.tensor([77, 4998], device="cuda")
    r = x.offs[1]
    x.logits[r].fill_(-inf)                           # nothing to choose from
    r = x.offs[2]
    x.logits[r].fill_(low)
    x.logits[r, 123] = 0.0                            # all else masked by the type's lowest value
    x.drafts[2, 0] = 123
    r = x.offs[3]
    x.logits[r, ::2] = math.nan                       # NaN is never chosen
    x.logits[r, 11] = inf                             # one infinite logit takes everything
    x.drafts[3, 0] = 12
    r = x.offs[4]
    x.logits[r].fill_(math.nan)
    r = x.offs[5]
    x.drafts[5, 0] = 9
    x.uniforms[5, 0] = 0.0
    x.logits[r, 9] = -inf                             # probability zero is refused even by u = 0
    acc, tok, probs = x.run(N)
    assert acc.tolist()[:5] == [1, 0, 1, 0, 0]
    assert tok.tolist()[0] == 4999 and tok.tolist()[1] == -1 and tok.tolist()[3] == 11 and tok.tolist()[4] == -1
    assert probs[0].tolist() == [1.0, 1.0, 0.0] and probs[1].tolist() == [0.0] * 3 and probs[3].tolist() == [1.0, 0, 0]
    assert float(probs[2, 0]) == 1.0
    assert int(acc[5]) == 0 and int(tok[5]) != 9
    want = R.verify_sampled(x.logits, x.cu, x.drafts, x.uniforms, x.noise, x.heat)
    assert torch.equal(acc, want[0]) and torch.equal(tok, want[1])


def test_verify_follows_the_target(N):
    # the first emitted token's frequencies against p, drafts drawn from q: 5 standard deviations
    B, V = 40000, 6
    g = torch.Generator(device="cuda").manual_seed(1)
    one = torch.randn(2, V, device="cuda", generator=g) * 1.5
    q = torch.softmax(torch.randn(V, device="cuda", generator=g) * 1.5, 0)
    drafts = torch.multinomial(q, B, replacement=True, generator=g)[:, None]
    p = torch.softmax(one[0].double(), 0).cpu()
    for probs in (q.expand(B, 1, V).contiguous(), None):
        acc, tok, _ = N.verify_sampled(one.repeat(B, 1), torch.arange(0, 2 * B + 1, 2, dtype=torch.int32, device="cuda"), drafts,
                                       torch.rand(B, 1, device="cuda", generator=g),
                                       torch.empty(B, V, device="cuda").exponential_(generator=g),
                                       torch.ones(B, device="cuda"), probs)
        first = torch.where(acc == 1, drafts[:, 0], tok)
        if probs is None:  # certain drafts: given the draft, what is emitted follows p too
            first = first[drafts[:, 0] == 2]
        f = torch.bincount(first, minlength=V).double().cpu() / first.numel()
        assert ((f - p).abs() <= 5 * torch.sqrt(p * (1 - p) / first.numel())).all(), (f, p)


def test_verify_streams(N):
    x = Drafts([4, 2, 0, 3], 151936, [0.8], seed=8, dtype=torch.bfloat16)
    want = x.run(N)
    streams = [torch.cuda.Stream() for _ in range(4)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    outs = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(x.run(N))
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(a, b) for a, b in zip(o, want))


def test_verify_graph(N):
    x = Drafts([4, 2, 0, 3], 20000, [0.8], seed=9, dtype=torch.bfloat16)
    x.run(N)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = x.run(N)
    for seed in (10, 11):
        y = Drafts([4, 2, 0, 3], 20000, [0.8], seed=seed, dtype=torch.bfloat16)
        for name in ("logits", "drafts", "uniforms", "noise"):
            getattr(x, name).copy_(getattr(y, name))
        graph.replay()
        x.check(got)


def test_verify_bad_rows_are_reported(N):
    from mod_b200.ops import check_status

    x = Drafts([2, 2], 100, [1.0], seed=3)
    x.cu = ints([0, 3, 60])
    acc, tok, probs = x.run(N)
    with pytest.raises(RuntimeError, match="out of bounds"):
        check_status()
    assert int(acc[1]) == 0 and int(tok[1]) == -1 and (probs[1] == 0).all()


def test_verify_refuses(N):
    x = Drafts([2, 2], 100, [1.0], seed=3, q_dtype=torch.float32)
    good = (x.logits, x.cu, x.drafts, x.uniforms, x.noise, x.heat, x.probs)
    for i, bad in ((0, x.logits.half()), (0, x.logits[:, ::2]), (0, x.logits.cpu()), (1, x.cu.long()), (1, x.cu[1:]),
                   (2, x.drafts.int()), (3, x.uniforms.double()), (3, x.uniforms[:1]), (4, x.noise[:, :50]),
                   (4, x.noise.cpu()), (5, x.heat[:1]), (6, x.probs[:, :1]), (6, x.probs.half())):
        args = list(good)
        args[i] = bad
        with pytest.raises(RuntimeError):
            N.verify_sampled(*args)
