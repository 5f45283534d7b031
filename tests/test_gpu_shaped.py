"""GPU tests of attention with shaped scores (lt_kv_attend_shaped) over f16,
Q8_0 and Q4_0 caches against softmax attention in 64 bits.

Tolerances as for plain attention (rtol 1e-4, atol 2e-5 for f32 outputs; f16
outputs add half a step, 2^-11): tanhf is within 2 ulp, so the cap moves a
score of magnitude up to 50 by at most 2 * 2^-24 * 50 * log2(e) < 1e-5 in the
exponent; the distance term is one f32 product and difference, off by at most
2^-24 of a magnitude of which only positions within ~25 of the largest score
weigh anything."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import _attn64 as A  # noqa: E402

from langtrain_studio_b200.kv import KvCache, KvError  # noqa: E402

pytestmark = pytest.mark.gpu
FORMATS = ["f16", "q8_0", "q4_0"]


@pytest.fixture(scope="module", autouse=True)
def _need_cuda():
    if not torch.cuda.is_available():
        pytest.fail("CUDA device required for -m gpu tests")


class Cache:
    def __init__(self, fmt, hkv, hd, hq, lens, rng, **kw):
        self.kv = KvCache(1, hkv, hd, 16 * sum((n + 15) // 16 for n in lens), n_heads=hq, max_seqs=len(lens),
                          max_batch=4096, kv_format=fmt, **kw)
        self.group, self.hq, self.hd, self.vals = hq // hkv, hq, hd, []
        for s, n in enumerate(lens):
            x = rng.standard_normal((2, n, hkv * hd)).astype(np.float32)
            cells = self.kv.append_batch(np.full(n, s), np.arange(n))
            self.kv.write(0, *cells, *(torch.from_numpy(a).cuda() for a in x))
            y = x.reshape(2, n, hkv, hd)
            if fmt == "f16":
                y = y.astype(np.float16).astype(np.float64)
            elif fmt == "q8_0":
                y = A.quant8(y)
            else:
                y = A.value4(*A.quant4(y))
            self.vals.append(y)

    def run(self, seqs, pos, q, out_dtype=torch.float32, **shape):
        """(out, reference) of the tokens; shape as attend_shaped's arguments."""
        dev = dict(shape)
        if shape.get("slopes") is not None:
            dev["slopes"] = torch.from_numpy(shape["slopes"]).cuda()
        out = self.kv.attend_shaped(0, q, seqs, pos, out_dtype=out_dtype, **dev)
        self.kv.check()
        ref = np.zeros((len(seqs), self.hq * self.hd))
        qn = q.float().cpu().numpy().reshape(len(seqs), self.hq, self.hd)
        for i, (s, p) in enumerate(zip(seqs, pos)):
            one = {k: (v[i] if k in ("first", "end") and v is not None else v) for k, v in shape.items()}
            k, v = self.vals[int(s)]
            ref[i] = A.attend(qn[i], k, v, int(p), self.group, self.kv.default_scale, **one).reshape(-1)
        return out, ref


def close(out, ref, out_dtype=torch.float32):
    half = out_dtype == torch.float16
    np.testing.assert_allclose(out.float().cpu().numpy(), ref, rtol=1e-4 + (2 ** -11 if half else 0),
                               atol=2e-5 + (2 ** -24 if half else 0))


def slopes_of(hq):
    return np.exp2(-8.0 * np.arange(1, hq + 1) / hq).astype(np.float32)


TERMS = {
    "nothing": dict(),
    "cap": dict(softcap=3.0),
    "cap50": dict(softcap=50.0),
    "window1": dict(window=1),
    "window": dict(window=37),
    "wide window": dict(window=100000),
    "bias": dict(slopes=True),
    "all": dict(softcap=20.0, window=130, slopes=True),
}


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("terms", sorted(TERMS))
@pytest.mark.parametrize("hd,hq,hkv", [(128, 32, 8), (64, 14, 2)])
def test_terms(fmt, terms, hd, hq, hkv):
    rng = np.random.default_rng(len(terms) + hd)
    lens = [1, 16, 17, 37, 300, 555]
    c = Cache(fmt, hkv, hd, hq, lens, rng)
    c.kv.set_min_tiles_per_warp(2)
    shape = dict(TERMS[terms])
    if shape.pop("slopes", False):
        shape["slopes"] = slopes_of(hq)
    for dtype in (torch.float32, torch.float16):
        q = torch.from_numpy(2 * rng.standard_normal((len(lens), hq * hd)).astype(np.float32)).cuda().to(dtype)
        out, ref = c.run(np.arange(len(lens)), np.array(lens) - 1, q, dtype, **shape)
        close(out, ref, dtype)
        if terms in ("nothing", "wide window"):
            plain = c.kv.attend(0, q, np.arange(len(lens)), np.array(lens) - 1, out_dtype=dtype)
            close(plain, ref, dtype)


@pytest.mark.parametrize("fmt", FORMATS)
def test_intervals(fmt):
    """Per-token intervals of packed documents with a bidirectional prefix:
    starts and ends inside blocks, one position, the whole sequence, empty."""
    rng = np.random.default_rng(4)
    hd, hq, hkv = 64, 8, 2
    c = Cache(fmt, hkv, hd, hq, [200, 35], rng)
    c.kv.set_min_tiles_per_warp(1)
    cases = [  # (seq, pos, first, end)
        (0, 199, 0, 200), (0, 199, 0, 199), (0, 50, 0, 200), (0, 50, 16, 32), (0, 50, 17, 31), (0, 50, 15, 16),
        (0, 50, 16, 17), (0, 50, 199, 200), (0, 50, 100, 100), (0, 50, 180, 3), (0, 0, 0, 1), (0, 0, 0, 0),
        (0, 120, 47, 121), (1, 34, 0, 35), (1, 34, 33, 35), (1, 3, 4, 4), (1, 3, 4294967295, 35), (0, 7, 5, 190),
    ]
    seqs, pos, first, end = (np.array(x) for x in zip(*cases))
    q = torch.from_numpy(rng.standard_normal((len(cases), hq * hd)).astype(np.float32)).cuda()
    for extra in (dict(), dict(softcap=5.0, slopes=slopes_of(hq)), dict(window=20)):
        out, ref = c.run(seqs, pos, q, first=first, end=end, **extra)
        close(out, ref)
        empty = [i for i, (s, p, f, e) in enumerate(cases) if f >= e]
        assert not out[empty].any()
    out, ref = c.run(seqs, pos, q, first=np.minimum(first, pos))  # end left to the causal default
    close(out, ref)


@pytest.mark.parametrize("fmt", FORMATS)
def test_prefix_chunk_over_512_tokens(fmt):
    """A chunk of 700 tokens whose first 100 positions see one another."""
    rng = np.random.default_rng(6)
    c = Cache(fmt, 1, 64, 4, [700], rng)
    pos = np.arange(700)
    q = torch.from_numpy(rng.standard_normal((700, 4 * 64)).astype(np.float32)).cuda()
    out, ref = c.run(np.zeros(700, int), pos, q, end=np.maximum(pos + 1, 100), slopes=slopes_of(4))
    close(out, ref)


@pytest.mark.parametrize("fmt", ["f16", "q8_0"])
def test_masked_cells_hold_inf_and_nan(fmt):
    """Inf and NaN rows before an interval, inside its first and last blocks
    and in blocks of their own never reach an output."""
    rng = np.random.default_rng(9)
    hd, n = 128, 100
    c = Cache(fmt, 2, hd, 8, [n], rng)
    bad = torch.full((1, 2 * hd), float("nan"), device="cuda")
    inf = torch.full((1, 2 * hd), float("inf"), device="cuda")
    blocks = c.kv.seq_blocks(0)
    for p in list(range(0, 37)) + [61, 62, 63, 90]:
        c.kv.write(0, [blocks[p // 16]], [p % 16], bad if p % 2 else inf, inf if p % 3 else bad)
    q = torch.from_numpy(rng.standard_normal((2, 8 * hd)).astype(np.float32)).cuda()
    first, end = np.array([37, 40]), np.array([61, 61])
    out, ref = c.run([0, 0], [99, 60], q, first=first, end=end)
    close(out, ref)
    out, ref = c.run([0, 0], [60, 60], q, window=20)
    close(out, ref)


def test_long_window_reads_few_blocks_and_merges():
    """A window deep in a long sequence, cut over several warps."""
    rng = np.random.default_rng(12)
    for fmt in FORMATS:
        c = Cache(fmt, 1, 128, 8, [4000], rng)
        q = torch.from_numpy(rng.standard_normal((1, 8 * 128)).astype(np.float32)).cuda()
        for tiles in (1, 8):
            c.kv.set_min_tiles_per_warp(tiles)
            out, ref = c.run([0], [3990], q, window=1500, softcap=30.0, slopes=slopes_of(8))
            close(out, ref)


def test_repeated_calls_are_bit_equal():
    rng = np.random.default_rng(15)
    c = Cache("q4_0", 4, 64, 16, [900, 30, 444], rng)
    q = torch.from_numpy(rng.standard_normal((3, 16 * 64)).astype(np.float32)).cuda()
    args = dict(softcap=9.0, window=500)
    a = c.kv.attend_shaped(0, q, [0, 1, 2], [899, 29, 443], **args)
    for _ in range(5):
        assert torch.equal(a, c.kv.attend_shaped(0, q, [0, 1, 2], [899, 29, 443], **args))


def test_refusals():
    rng = np.random.default_rng(1)
    c = Cache("f16", 1, 64, 4, [20], rng)
    q = torch.zeros((1, 256), device="cuda")
    ok = c.kv.attend_shaped(0, q, [0], [19])
    for kw, err in [(dict(softcap=-1.0), KvError), (dict(softcap=float("nan")), KvError),
                    (dict(softcap=float("inf")), KvError), (dict(softcap=1e-45), KvError), (dict(end=[21]), KvError), (dict(window=-1), ValueError),
                    (dict(first=[0, 0]), ValueError), (dict(end=[-1]), ValueError),
                    (dict(slopes=torch.zeros(4)), ValueError), (dict(slopes=torch.zeros(3, device="cuda")), ValueError),
                    (dict(slopes=torch.zeros(4, device="cuda", dtype=torch.float16)), TypeError)]:
        with pytest.raises(err):
            c.kv.attend_shaped(0, q, [0], [19], **kw)
    for args, err in [((0, q, [0], [20]), KvError), ((1, q, [0], [19]), KvError), ((0, q, [1], [0]), KvError),
                      ((0, q[:, ::2], [0], [19]), ValueError), ((0, q.cpu(), [0], [19]), ValueError),
                      ((0, q, [0], [19, 19]), ValueError)]:
        with pytest.raises(err):
            c.kv.attend_shaped(*args)
    assert c.kv.attend_shaped(0, q[:0], [], []).shape == (0, 256)
    assert torch.equal(ok, c.kv.attend_shaped(0, q, [0], [19]))


def test_large_caps():
    """A cap that no score comes near leaves plain attention (tanhf keeps its
    relative accuracy near 0).  Above 1e30 it is refused: s / softcap would fall
    among the subnormals and softcap * log2(e) pass the largest f32."""
    rng = np.random.default_rng(77)
    for fmt in FORMATS:
        c = Cache(fmt, 2, 128, 8, [40], rng)
        q = torch.from_numpy(rng.standard_normal((1, 8 * 128)).astype(np.float32)).cuda()
        for cap in (1e4, 1e15, 1e30):
            out, ref = c.run([0], [39], q, softcap=cap)
            close(out, ref)
        for cap in (1.1e30, 3e38):
            with pytest.raises(KvError, match="softcap"):
                c.run([0], [39], q, softcap=cap)


@pytest.mark.parametrize("hd,hq,hkv", [(128, 32, 8), (64, 16, 16), (64, 6, 2)])
@pytest.mark.parametrize("terms", ["nothing", "window", "all", "documents", "prefix"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_chunks_over_the_4_bit_cache(hd, hq, hkv, terms, dtype):
    """Prefill chunks with shaped scores, which the tensor-core pass attends whole
    over the blocks of their intervals: windows and documents that start inside a
    block, empty intervals (alone in a 128-row tile too), ends past the token."""
    rng = np.random.default_rng(hd + hq + len(terms))
    lens = [300, 61, 700, 8]
    c = Cache("q4_0", hkv, hd, hq, lens, rng)
    seqs = np.concatenate([np.full(260, 0), np.full(61, 1), np.full(330, 2), np.full(8, 3)])
    pos = np.concatenate([np.arange(40, 300), np.arange(61), np.arange(370, 700), np.arange(8)])
    shape = {}
    if terms == "window":
        shape = dict(window=50)
    elif terms == "all":
        shape = dict(softcap=20.0, window=130, slopes=slopes_of(hq))
    elif terms == "documents":
        first = pos // 90 * 90
        end = pos + 1
        first[(seqs == 2) & (pos < 520)] = 600  # empty: they start past their end
        shape = dict(first=first, end=end, slopes=slopes_of(hq))
    elif terms == "prefix":
        shape = dict(end=np.minimum(np.array(lens)[seqs], np.maximum(pos + 1, 200)), softcap=5.0)
    q = torch.from_numpy(rng.standard_normal((seqs.size, hq * hd)).astype(np.float32)).cuda().to(dtype)
    c0 = c.kv.cascade_launches()
    out, ref = c.run(seqs, pos, q, dtype, **shape)
    close(out, ref, dtype)
    if hkv > 2:  # enough tiles for the device (groups of 3 on 2 heads leave most of it free)
        assert c.kv.cascade_launches() == c0 + 1
    if terms == "documents":
        assert not out[torch.from_numpy((seqs == 2) & (pos < 520)).cuda()].any()
    # the same tokens in another order give the same rows
    mix = np.concatenate([rng.permutation(260) + 260 * 0, 321 + rng.permutation(330), 260 + rng.permutation(61)])
    part = {k: (v[mix] if k in ("first", "end") else v) for k, v in shape.items()}
    out2, ref2 = c.run(seqs[mix], pos[mix], q[torch.from_numpy(mix).cuda()].contiguous(), dtype, **part)
    close(out2, ref2, dtype)


def test_short_chunks_over_the_4_bit_cache():
    """Chunks whose intervals are short are attended whole however few they are."""
    rng = np.random.default_rng(5)
    c = Cache("q4_0", 1, 128, 4, [2000], rng)
    pos = np.arange(1500, 1520)
    q = torch.from_numpy(rng.standard_normal((20, 512)).astype(np.float32)).cuda()
    for window in (1, 16, 17, 60, 1000):
        c0 = c.kv.cascade_launches()
        out, ref = c.run(np.zeros(20, int), pos, q, window=window)
        close(out, ref)
        assert c.kv.cascade_launches() == c0 + (window < 1000)


@pytest.mark.parametrize("fmt", ["f16", "q8_0"])
def test_large_calls_with_changing_intervals(fmt):
    """Calls of more than 512 tokens, whose tokens and intervals are staged apart:
    the same tokens again and again with other intervals (global and windowed
    layers, packed documents), more calls than the staging has places."""
    rng = np.random.default_rng(23)
    c = Cache(fmt, 1, 64, 2, [160] * 4, rng)
    seqs, pos = np.repeat(np.arange(4), 144), np.tile(np.arange(16, 160), 4)
    q = torch.from_numpy(rng.standard_normal((seqs.size, 2 * 64)).astype(np.float32)).cuda()
    outs = []
    for call in range(20):
        first = (np.arange(seqs.size) + 5 * call) % 16
        outs.append((c.kv.attend_shaped(0, q, seqs, pos, first=first), first))
    c.kv.check()
    for out, first in outs:
        ref = np.zeros((seqs.size, 128))
        for i, (s, p) in enumerate(zip(seqs, pos)):
            ref[i] = A.attend(q[i].cpu().numpy().reshape(2, 64), *c.vals[s], int(p), 2, c.kv.default_scale,
                              first=first[i]).reshape(-1)
        close(out, ref)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("length", [100, 128, 190, 1100])
def test_warps_of_the_pass_run_apart(hd, length):
    """Prompts through the tensor-core pass whose rows move their maximum at every
    step in some warps (steep slopes) and never in others (an interval that ends
    early, no q), over 2, 3 and many steps of 64 positions: a warp that has nothing
    to rescale runs ahead of one that has.  Every repetition gives the same bits."""
    rng = np.random.default_rng(hd + length)
    seqs_n, chunk, hq, hkv = 4, 100, 32, 8
    c = Cache("q4_0", hkv, hd, hq, [length] * seqs_n, rng)
    seqs = np.repeat(np.arange(seqs_n), chunk)
    pos = np.tile(np.arange(length - chunk, length), seqs_n)
    end = pos + 1
    early = np.tile(np.arange(chunk) % 16 < 8, seqs_n)  # 8 tokens are the 32 rows of a warp
    end[early & (seqs < 2)] = 17
    q = rng.standard_normal((seqs.size, hq * hd)).astype(np.float32)
    q[early & (seqs >= 2)] = 0
    q[~early] *= 3
    slopes = np.where(np.arange(hq) % 4 == 0, 0.0, 1.0).astype(np.float32)
    c0 = c.kv.cascade_launches()
    qd = torch.from_numpy(q).cuda()
    out, ref = c.run(seqs, pos, qd, end=end, slopes=slopes)
    assert c.kv.cascade_launches() == c0 + 1
    # Where an interval ends far before its token, every distance in it is near D =
    # pos: slope * D * log2(e) < 2^11 has a spacing of 2^-13 in f32, its product and
    # the difference round by half of that each, so a weight is off by a factor of
    # 2^(2^-13) at most, and an output by 2 * ln(2) * 2^-13 * max|v|.  The other rows
    # keep the bar above: what weighs in them lies near the token.
    far = torch.from_numpy(end == 17)
    close(out[~far], ref[~far.numpy()])
    most = max(np.abs(v).max() for _, v in c.vals)
    spacing = np.spacing(np.float32(length * np.log2(np.e)))
    assert np.abs(out[far].cpu().numpy() - ref[far.numpy()]).max() <= 2e-5 + 2 * np.log(2) * spacing * most
    sd = torch.from_numpy(slopes).cuda()
    again = [c.kv.attend_shaped(0, qd, seqs, pos, end=end, slopes=sd) for _ in range(100)]
    c.kv.check()
    for a in again:
        assert torch.equal(a, out)
