"""The limits of the kernels behind sampling several continuations of one prompt: launch sizes at the edge of what a CTA
may have without asking, sums past 32 bits, offsets and temperatures at the ends of their types, refused arguments."""
import math
import os
import subprocess
import sys

import pytest
import torch

from mod_b200.ops import reference as R
from tests.test_shared_sampling_gpu import PAGE, Batch, Drafts, ints, seqs

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


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


def alone(code, *args):
    """Runs ``code`` in a process of its own, where no earlier call has asked for more shared memory."""
    r = subprocess.run([sys.executable, "-c", code, *map(str, args)], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-1500:]


PLAN = """
import sys, torch
from mod_b200.ops import check_status, native as N
B, G = map(int, sys.argv[1:])
i = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
k = torch.randn(2, 1, 16, 64, device="cuda").bfloat16()
v = torch.randn(2, 1, 64, 16, device="cuda").bfloat16()
q = torch.randn(B, 1, 64, device="cuda").bfloat16()
tables, ctx = torch.ones(B, 1, dtype=torch.int32, device="cuda"), torch.ones(B, dtype=torch.int32, device="cuda")
offs = i(list(range(B + 1))) if G == B else i([0, B])
p = N.attn_shared_plan(tables, ctx, offs, i([0] * G), B, 1, 1, 64)
out = N.attn_shared(q, k, v, tables, p)
assert torch.equal(out, v[1, :, :, 0].expand(B, 1, 64))   # one key: its value
check_status()
"""


# Shared memory: 4 (4 G + 3 B + 8) bytes beside 132 static ones; 48 KB is what a launch has without asking.
@pytest.mark.parametrize("B,G", [(1749, 1749), (1750, 1750), (1754, 1754), (1755, 1755), (4082, 1), (4092, 1)])
def test_plan_at_48_kb(B, G, cuda):
    alone(PLAN, B, G)


COMPACT = """
import sys, torch
from mod_b200.ops import check_status, native as N
pages = int(sys.argv[1])
k = [torch.zeros(pages, 1, 16, 8, dtype=torch.bfloat16, device="cuda")]
v = [torch.zeros(pages, 1, 8, 16, dtype=torch.bfloat16, device="cuda")]
k[0][pages - 1], v[0][pages - 1] = 1.0, 2.0
one = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
tables, remap, live = N.kv_compact(k, v, one([[pages - 1]]), one([16]))
assert tables.tolist() == [[0]] and int(live) == 1 and int(remap[pages - 1]) == 0
assert (k[0][0] == 1).all() and (v[0][0] == 2).all()
check_status()
"""


# A bit a page beside 128 static bytes.
@pytest.mark.parametrize("pages", [392_192, 392_193, 393_216, 393_217])
def test_compact_at_48_kb(pages, cuda):
    alone(COMPACT, pages)


def plan_only(N, B, pages, heads):
    """The schedule of B sequences of `pages` full pages, a token each, on one KV head; tables are not read for it."""
    tables = torch.zeros(1, 1, dtype=torch.int32, device="cuda").expand(B, pages)
    ctx = torch.full((B,), pages * PAGE, dtype=torch.int32, device="cuda")
    return N.attn_shared_plan(tables, ctx, ints(range(B + 1)), ints([0] * B), B, heads, 1, 64)


def test_plan_counts_pages_past_32_bits(N):
    # 8192 sequences x 4 row tiles x 65536 pages = 2^31: a schedule like any other
    plan_only(N, 8192, 65536, 64)
    torch.cuda.synchronize()
    from mod_b200.ops import check_status

    check_status()


def test_plan_costs_past_32_bits_are_reported(N):
    # 8192 units of 131072 key tiles and more: their cost does not fit the schedule's sums, which is said
    from mod_b200.ops import check_status

    plan_only(N, 8192, 524288 + 64, 128)
    with pytest.raises(RuntimeError, match="out of bounds"):
        check_status()
    plan_only(N, 4000, 524288 + 64, 128)
    torch.cuda.synchronize()
    check_status()


@pytest.mark.parametrize("cu", [[0, 3, 2 ** 31 - 1], [0, 2 ** 31 - 2, -2 ** 31 + 1], [0, -2 ** 31, 2 ** 31 - 1],
                                [2 ** 31 - 1, -2 ** 31, 6], [0, 6, 6], [0, 0, 6]], ids=str)
def test_verify_offsets_at_the_ends_are_reported(N, cu):
    from mod_b200.ops import check_status

    x = Drafts([2, 2], 100, [1.0], seed=3)
    want = x.run(N)
    x.cu = ints(cu)
    got = x.run(N)
    with pytest.raises(RuntimeError, match="out of bounds"):
        check_status()
    for b in range(2):
        lo, hi = cu[b], cu[b + 1]
        if (lo, hi) == (x.offs[b], x.offs[b + 1]):
            assert all(torch.equal(g[b], w[b]) for g, w in zip(got, want))
        else:
            assert int(got[0][b]) == 0 and int(got[1][b]) == -1 and (got[2][b] == 0).all()


def test_no_heads_are_refused(N):
    for heads in (0, -8):
        with pytest.raises(RuntimeError, match="heads"):
            N.attn_shared_plan(ints([[0]]), ints([1]), ints([0, 1]), ints([0]), 1, heads, 2, 64)
    b = Batch([(0, seqs(3))], 2, 2, 64)
    p = b.plan(N)
    p.q_shape = torch.Size((1, 0, 64))
    with pytest.raises(RuntimeError, match="heads"):
        N.attn_shared(b.q[:, :0], b.k, b.v, b.tables, p)


def test_attn_shared_buffers_off_their_alignment_are_refused(N):
    b = Batch([(40, seqs(3, 20))], 8, 2, 128)
    p = b.plan(N)
    C, out = N._C(), torch.empty_like(b.q)
    ws = torch.empty(p.ws_elems + 8, dtype=torch.float32, device="cuda")
    buf = torch.empty(p.buf.numel() + 4, dtype=torch.int32, device="cuda")
    scale = 1 / math.sqrt(128)
    for off in (1, 2, 4):
        with pytest.raises(RuntimeError, match="aligned"):
            C.attn_shared(b.q, b.k, b.v, b.tables, 1, p.buf, ws[off:], out, scale)
    for off in (1, 2, 3):
        with pytest.raises(RuntimeError, match="aligned"):
            C.attn_shared(b.q, b.k, b.v, b.tables, 1, buf[off:], ws, out, scale)
        with pytest.raises(RuntimeError, match="aligned"):
            C.attn_shared_plan(b.tables, ints(b.ctx), ints(b.offs), ints(b.shared), None, 2, 8, 2, 128, buf[off:])
    for plan, work in ((p.buf.repeat_interleave(2)[::2], ws), (p.buf, torch.cat([ws, ws])[::2])):
        with pytest.raises(RuntimeError, match="contiguous"):
            C.attn_shared(b.q, b.k, b.v, b.tables, 1, plan, work, out, scale)
    C.attn_shared(b.q, b.k, b.v, b.tables, 1, p.buf, ws[8:], out, scale)
    b.check(out)


HEATS = [1e-45, 1e-40, 4e-39, 2 ** -126, 1e-30, 1e30, torch.finfo(torch.float32).max, math.inf]


@pytest.mark.parametrize("q_dtype", [None, torch.float32])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_verify_temperatures_at_the_ends(N, dtype, q_dtype):
    # all of the probability on the largest logit at one end, the same for every id at the other
    x = Drafts([2] * len(HEATS), 1000, HEATS, seed=21, dtype=dtype, q_dtype=q_dtype)
    x.check(x.run(N))


def test_verify_infinite_temperature_and_masks(N):
    # masked ids stay out however hot the rest is
    x = Drafts([1, 1, 0], 1000, [math.inf, torch.finfo(torch.float32).max, math.inf], seed=22)
    x.logits[:, 100:] = -math.inf
    x.logits[:, 100] = torch.finfo(torch.float32).min
    x.drafts[:] = 500
    acc, tok, probs = x.run(N)
    want = R.verify_sampled(x.logits, x.cu, x.drafts, x.uniforms, x.noise, x.heat)
    assert torch.equal(acc, want[0]) and torch.equal(tok, want[1])
    assert acc.tolist() == [0, 0, 0] and 0 <= int(tok.min()) and int(tok.max()) <= 100
    assert (probs[:, 0] > 0).all() and torch.allclose(probs, want[2], rtol=2 ** -18, atol=0)


def fine_errors(b, out):
    """Largest errors over sum(p |v|) beyond the output's last rounding: of ``out``, and of what weights rounded to one
    bf16 would give."""
    T, Hq, D = b.q.shape
    rep, worst = Hq // b.k.shape[1], [0.0, 0.0]
    for s, c in enumerate(b.ctx):
        t0, t1 = b.cu[s], b.cu[s + 1]
        k = R.gather_kv(b.k, b.tables[s], c).double().repeat_interleave(rep, 1)
        v = R.gather_v(b.v, b.tables[s], c).double().repeat_interleave(rep, 1)
        x = torch.einsum("qhd,nhd->hqn", b.q[t0:t1].double(), k) / math.sqrt(D)
        seen = torch.arange(c, device=x.device)[None, :] <= c - (t1 - t0) + torch.arange(t1 - t0, device=x.device)[:, None]
        x = x.masked_fill(~seen[None], -math.inf)
        p = torch.softmax(x, -1)
        o, size = torch.einsum("hqn,nhd->qhd", p, v), torch.einsum("hqn,nhd->qhd", p, v.abs())
        e = torch.exp(x - x.amax(-1, keepdim=True))
        one = torch.einsum("hqn,nhd->qhd", e.bfloat16().double() / e.sum(-1, keepdim=True), v).bfloat16()
        for i, got in enumerate((out[t0:t1], one)):
            worst[i] = max(worst[i], float((((got.double() - o).abs() - 2 ** -8 * o.abs()) / size).max()))
    return worst


# Values are 1 or -1, so that sums of them cancel and the output's own rounding, 2^-8 of it, hides little.  A key's weight as
# one bf16 is off by up to 2^-8 of itself; as two bf16 terms by 2^-16, and the exponentials and sums in 32 bits add a few
# 2^-22 for scores of a few units.
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("groups", [[(0, [(40, 1), (33, 4)])], [(0, [(150, 90), (130, 130)])], [(256, [(1, 1)] * 4)],
                                    [(112, [(1, 1)] * 70)]], ids=["few rows", "many rows", "prefix", "prefix of part tiles"])
def test_weights_keep_sixteen_bits(N, D, groups):
    b = Batch(groups, 8, 2, D, seed=31, q_scale=1.0)
    b.v.copy_(torch.where(b.v > 0, 1.0, torch.where(b.v <= 0, -1.0, b.v.float())))  # NaN stays where no token is
    mine, one_term = fine_errors(b, N.attn_shared(b.q, b.k, b.v, b.tables, b.plan(N)))
    assert mine <= 2 ** -15 < 2 ** -14 < one_term
