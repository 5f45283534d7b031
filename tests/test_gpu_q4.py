"""GPU tests of the 4-bit cache (include/lt_kv.h, LT_KV_Q4_0) through the C ABI.

Codes and scales are bit-exact against a 64-bit restatement of the format on
every write path (f32, f16, fused append, copy-on-write, compaction); values
read back exactly.  Attention is compared with softmax attention in 64 bits
over the cached values.

Tolerances.  Cached values are f16s exactly and q and the weights are carried
as f16 value + residual (relative error 2^-22 each); 2^x on the SFU is within
2^-22; scores and sums are f32.  A score of magnitude up to 16 with 128 f32
additions moves by at most ~128 * 2^-24 * 16 * log2(e) / sqrt(128) (random
signs) ~ 2e-5 in the exponent for single positions, which averages out over
the sum; rtol 1e-4 and atol 2e-5 (the other formats' bar) cover it.  f16
outputs add half a step, 2^-11 relative."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import _attn64 as A  # noqa: E402

from langtrain_studio_b200.kv import BLOCK, KvCache, KvError  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_cuda():
    if not torch.cuda.is_available():
        pytest.fail("CUDA device required for -m gpu tests")


class Twin:
    """A Q4_0 KvCache and the values it must hold, per sequence."""

    def __init__(self, hkv, hd, tokens, hq=None, layers=1, max_seqs=8, **kw):
        self.kv = KvCache(layers, hkv, hd, tokens, n_heads=hq or hkv, max_seqs=max_seqs, kv_format="q4_0", **kw)
        self.hkv, self.hd, self.hq, self.layers = hkv, hd, hq or hkv, layers
        self.rows = {}  # (layer, seq) -> list of (kc, kd, vc, vd) rows

    def add(self, layer, seq, k, v):
        rows = self.rows.setdefault((layer, seq), [])
        for a, b in zip(k.reshape(-1, self.hkv, self.hd), v.reshape(-1, self.hkv, self.hd)):
            rows.append((*A.quant4(a), *A.quant4(b)))

    def draw(self, n, rng, dtype=np.float32):
        return tuple((rng.standard_normal((n, self.hkv * self.hd)) * g).astype(dtype) for g in (1.5, 1.0))

    def fill(self, seq, upto, rng, dtype=np.float32):
        n0 = self.kv.len(seq)
        if upto <= n0:
            return
        pos = np.arange(n0, upto)
        cells = self.kv.append_batch(np.full(pos.size, seq), pos)
        for layer in range(self.layers):
            k, v = self.draw(pos.size, rng, dtype)
            self.kv.write(layer, *cells, torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda())
            self.add(layer, seq, k, v)

    def values(self, layer, seq):
        """(K, V) [len, hkv, hd] f64."""
        rows = self.rows[(layer, seq)][: self.kv.len(seq)]
        return (np.stack([A.value4(r[0], r[1]) for r in rows]), np.stack([A.value4(r[2], r[3]) for r in rows]))

    def check(self, layer, seq):
        """Codes and scales in the pool, through the table, bit for bit."""
        n = self.kv.len(seq)
        kc, vc, kd, vd = self.kv.pool_reference_layout(layer)
        blocks = self.kv.seq_blocks(seq)
        for i, (rk, dk, rv, dv) in enumerate(self.rows[(layer, seq)][:n]):
            b, s = blocks[i // BLOCK], i % BLOCK
            assert np.array_equal(kc[b, s], rk.reshape(-1)), (seq, i)
            assert np.array_equal(vc[b, s], rv.reshape(-1)), (seq, i)
            assert np.array_equal(kd[b, s].view(np.float16).astype(np.float64), dk.reshape(-1)), (seq, i)
            assert np.array_equal(vd[b, s].view(np.float16).astype(np.float64), dv.reshape(-1)), (seq, i)
        kr, vr = self.kv.rows(layer, seq, n)
        K, V = self.values(layer, seq)
        assert np.array_equal(kr.cpu().numpy().astype(np.float64).reshape(K.shape), K)
        assert np.array_equal(vr.cpu().numpy().astype(np.float64).reshape(V.shape), V)

    def attend_ref(self, layer, seqs, pos, q):
        out = np.zeros((len(seqs), self.hq * self.hd))
        cache = {}
        for i, (s, p) in enumerate(zip(seqs, pos)):
            if s not in cache:
                cache[s] = self.values(layer, s)
            K, V = cache[s]
            out[i] = A.attend(q[i].reshape(self.hq, self.hd), K, V, int(p), self.hq // self.hkv,
                              self.kv.default_scale).reshape(-1)
        return out


def close(out, ref, out_dtype=torch.float32):
    half = out_dtype == torch.float16
    np.testing.assert_allclose(out.float().cpu().numpy(), ref, rtol=1e-4 + (2 ** -11 if half else 0),
                               atol=2e-5 + (2 ** -24 if half else 0))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_write_is_bit_exact(hd, dtype):
    rng = np.random.default_rng(hd)
    t = Twin(4, hd, 16 * 20, layers=2, max_seqs=4)
    for s, n in enumerate([1, 17, 40, 100]):
        t.fill(s, n, rng, dtype)
    for s in range(4):
        for layer in range(2):
            t.check(layer, s)


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_write_borders_and_odd_values(dtype):
    """Values on and next to the code borders, ties of the two extremes, zeros,
    subnormals, saturation, Inf and NaN."""
    rng = np.random.default_rng(1)
    t = Twin(2, 64, 16 * 4, max_seqs=1)
    rows = []
    for sign in (1.0, -1.0):
        for d in (0.375, 1.0, 0.0078125, 2.0 ** -24, 3 * 2.0 ** -20, 300.0):
            steps = (np.arange(32) % 17 - 8.5)  # k + 1/2: exactly between two codes
            x = steps * d
            x[0] = -8 * d
            with np.errstate(over="ignore"):
                near = np.nextafter(x.astype(dtype), np.array(np.inf if sign > 0 else -np.inf, dtype))
            rows.append(np.concatenate([sign * x, sign * near.astype(np.float64), sign * 0.99 * x, rng.standard_normal(32)]))
    both = np.zeros(128)
    both[[3, 40, 70, 100]], both[[9, 35, 90, 110]] = 5.0, -5.0  # both signs reach the largest magnitude
    rows += [both, np.zeros(128), np.full(128, 1e-7), np.full(128, 30000.0), -np.linspace(1, 65000, 128)]
    odd = rng.standard_normal(128)
    odd[5], odd[37], odd[70], odd[71] = np.nan, np.inf, -np.inf, np.nan
    rows += [odd, np.full(128, np.nan), np.full(128, np.inf)]
    with np.errstate(over="ignore"):
        k = np.stack(rows).astype(dtype)
    v = k[::-1].copy()
    cells = t.kv.append_batch(np.zeros(len(k)), np.arange(len(k)))
    t.kv.write(0, *cells, torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda())
    t.add(0, 0, k, v)
    t.check(0, 0)
    # values read back and written again keep their codes
    kr, vr = t.kv.read(0, *cells)
    t.kv.write(0, *cells, kr, vr)
    K, V = t.values(0, 0)
    k2, v2 = t.kv.read(0, *cells, dtype=torch.float32)
    assert np.array_equal(k2.cpu().numpy().reshape(K.shape), K) and np.array_equal(v2.cpu().numpy().reshape(V.shape), V)


def test_writes_of_one_block_keep_their_neighbours():
    """Single rows in any slot order: each write changes its own slot alone."""
    rng = np.random.default_rng(2)
    t = Twin(3, 128, 64, max_seqs=1)
    t.fill(0, 40, rng)
    blocks = t.kv.seq_blocks(0)
    for p in [39, 0, 8, 7, 15, 16, 24, 31, 3, 11]:
        k, v = t.draw(1, rng)
        t.kv.write(0, [blocks[p // 16]], [p % 16], torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda())
        new = (A.quant4(k.reshape(3, 128)), A.quant4(v.reshape(3, 128)))
        t.rows[(0, 0)][p] = (*new[0], *new[1])
    t.check(0, 0)


ATT_CASES = [
    # (head_dim, n_heads, n_kv_heads, lens)
    (128, 32, 8, [1, 15, 16, 17, 200]),
    (128, 64, 8, [513, 1100]),
    (64, 32, 4, [31, 192, 64]),
    (128, 8, 8, [2049, 3]),      # group 1
    (64, 12, 4, [77, 300]),      # group 3
    (128, 10, 2, [65, 700]),     # group 5
    (64, 14, 2, [48, 333]),      # group 7
]


@pytest.mark.parametrize("hd,hq,hkv,lens", ATT_CASES)
@pytest.mark.parametrize("q_dtype,out_dtype,min_tiles", [(torch.float32, torch.float32, 8),
                                                         (torch.float16, torch.float16, 8),
                                                         (torch.float16, torch.float32, 2),
                                                         (torch.float32, torch.float32, 1)])
def test_attention(hd, hq, hkv, lens, q_dtype, out_dtype, min_tiles):
    rng = np.random.default_rng(hd + hq + len(lens))
    t = Twin(hkv, hd, 16 * (sum((n + 15) // 16 for n in lens)), hq, max_seqs=len(lens), max_batch=2100)
    t.kv.set_min_tiles_per_warp(min_tiles)
    for s, n in enumerate(lens):
        t.fill(s, n, rng)
    seqs, pos = np.arange(len(lens)), np.array(lens) - 1
    q = torch.from_numpy(rng.standard_normal((len(lens), hq * hd)).astype(np.float32)).cuda().to(q_dtype)
    out = t.kv.attend(0, q, seqs, pos, out_dtype=out_dtype)
    t.kv.check()
    close(out, t.attend_ref(0, seqs, pos, q.float().cpu().numpy()), out_dtype)


@pytest.mark.parametrize("gain", [1e-6, 30.0, 3e4])
def test_attention_of_small_and_large_q(gain):
    """q far below and above 1 keeps its 22 bits (rows are scaled by a power of
    two); the scale argument brings the scores back to ordinary ones."""
    rng = np.random.default_rng(5)
    t = Twin(2, 128, 16 * 20, 8, max_seqs=1)
    t.fill(0, 300, rng)
    q = (rng.standard_normal((1, 8 * 128)) * gain).astype(np.float32)
    out = t.kv.attend(0, torch.from_numpy(q).cuda(), [0], [299], scale=t.kv.default_scale / gain)
    K, V = t.values(0, 0)
    scale = float(np.float32(t.kv.default_scale / gain))
    ref = A.attend(q.reshape(8, 128), K, V, 299, 4, scale).reshape(1, -1)
    close(out, ref)


def test_prefill_chunk_and_repeated_tokens():
    """Several tokens of one sequence, the same token twice, lengths that end
    inside a block, and more than 512 tokens in a call."""
    rng = np.random.default_rng(8)
    t = Twin(2, 64, 16 * 64, 8, max_seqs=3, max_batch=1024)
    for s, n in enumerate([333, 40, 1]):
        t.fill(s, n, rng)
    seqs = np.concatenate([np.zeros(100), np.ones(40), [2, 2, 0, 0]]).astype(np.int64)
    pos = np.concatenate([np.arange(233, 333), np.arange(40), [0, 0, 5, 5]]).astype(np.int64)
    seqs, pos = np.concatenate([seqs, np.zeros(460, np.int64)]), np.concatenate([pos, rng.integers(0, 333, 460)])
    q = rng.standard_normal((seqs.size, 8 * 64)).astype(np.float32)
    out = t.kv.attend(0, torch.from_numpy(q).cuda(), seqs, pos)
    t.kv.check()
    close(out, t.attend_ref(0, seqs, pos, q))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("kv_dtype", [np.float32, np.float16])
def test_fused_append(hd, kv_dtype):
    """Decode steps through write_attend keep the pool bit-exact, and equal
    write followed by attend."""
    rng = np.random.default_rng(hd)
    hkv, hq = 4, 16
    t = Twin(hkv, hd, 16 * 40, hq, max_seqs=4)
    for s, n in enumerate([3, 30, 64, 100]):
        t.fill(s, n, rng)
    for _ in range(20):
        seqs = np.arange(4)
        pos = np.array([t.kv.len(s) for s in seqs])
        b, sl = t.kv.append_batch(seqs, pos)
        k, v = t.draw(4, rng, kv_dtype)
        for s in seqs:
            t.add(0, int(s), k[s], v[s])
        q = rng.standard_normal((4, hq * hd)).astype(np.float32)
        kd, vd, qd = (torch.from_numpy(x).cuda() for x in (k, v, q))
        out = t.kv.write_attend(0, b, sl, kd, vd, qd, seqs, pos)
        close(out, t.attend_ref(0, seqs, pos, q))
    assert torch.equal(out, t.kv.attend(0, qd, seqs, pos))
    for s in range(4):
        t.check(0, s)
    t.kv.check()


def test_copy_on_write_compaction_and_stale_blocks():
    rng = np.random.default_rng(7)
    t = Twin(2, 64, 16 * 90, 8, layers=2, max_seqs=12)
    t.fill(0, 200, rng)
    for s in range(1, 10):
        t.kv.share(0, s, 150 + s)
        for layer in range(2):
            t.rows[(layer, s)] = list(t.rows[(layer, 0)][: 150 + s])
        t.fill(s, 170 + 3 * s, rng)
    t.kv.truncate(0, 0)
    t.kv.truncate(4, 0)
    assert t.kv.compact() > 0
    t.fill(11, 21, rng)  # reuses freed blocks: stale codes past slot 5 of its last one
    seqs = np.array([1, 2, 3, 5, 6, 7, 8, 9, 11])
    pos = np.array([t.kv.len(int(s)) - 1 for s in seqs])
    q = rng.standard_normal((9, 8 * 64)).astype(np.float32)
    for layer in range(2):
        for s in (1, 5, 9, 11):
            t.check(layer, s)
        close(t.kv.attend(layer, torch.from_numpy(q).cuda(), seqs, pos), t.attend_ref(layer, seqs, pos, q))
    t.kv.check()


@pytest.mark.parametrize("hd,hq,hkv", [(128, 32, 8), (64, 8, 2), (128, 16, 2), (64, 5, 1)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_prefix_pass(hd, hq, hkv, dtype):
    """Prefill chunks and sequences on a shared prefix: the shared blocks go
    through the tensor-core pass over expanded tiles.  Its scores and sums are
    f32 with q and the weights as value + residual, like the other path's."""
    rng = np.random.default_rng(hd + hq)
    t = Twin(hkv, hd, 16 * 200, hq, max_seqs=14, max_batch=1024)
    t.fill(0, 333, rng)
    t.fill(1, 70, rng)
    for s in range(2, 13):
        t.kv.share(1, s, 70)
        t.rows[(0, s)] = list(t.rows[(0, 1)][:70])
        t.fill(s, 71 + 5 * (s % 4), rng)
    t.fill(13, 40, rng)
    # a chunk of sequence 0, eleven members of the shared prefix, one other
    seqs = np.concatenate([np.zeros(150), np.arange(2, 13), [13]]).astype(np.int64)
    pos = np.concatenate([np.arange(183, 333), [t.kv.len(s) - 1 for s in range(2, 13)], [39]]).astype(np.int64)
    q = torch.from_numpy(rng.standard_normal((seqs.size, hq * hd)).astype(np.float32)).cuda().to(dtype)
    ref = t.attend_ref(0, seqs, pos, q.float().cpu().numpy())
    c0 = t.kv.cascade_launches()
    close(t.kv.attend(0, q, seqs, pos, out_dtype=dtype), ref, dtype)
    assert t.kv.cascade_launches() == c0 + 1
    t.kv.set_cascade(0)
    close(t.kv.attend(0, q, seqs, pos, out_dtype=dtype), ref, dtype)
    assert t.kv.cascade_launches() == c0 + 1
    t.kv.check()


def test_long_sequence_two_level_merge():
    """One long sequence cut over many warps, each range a few tiles."""
    rng = np.random.default_rng(11)
    n = 16 * 700 + 5
    t = Twin(1, 128, n + 16, 8, max_seqs=1, max_batch=n)
    k, v = t.draw(n, rng)
    cells = t.kv.append_batch(np.zeros(n), np.arange(n))
    t.kv.write(0, *cells, torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda())
    K, V = (A.value4(*A.quant4(x.reshape(n, 1, 128))) for x in (k, v))
    q = rng.standard_normal((1, 8 * 128)).astype(np.float32)
    ref = A.attend(q.reshape(8, 128), K, V, n - 1, 8, t.kv.default_scale).reshape(1, -1)
    for tiles in (1, 8, 40):
        t.kv.set_min_tiles_per_warp(tiles)
        close(t.kv.attend(0, torch.from_numpy(q).cuda(), [0], [n - 1]), ref)
    t.kv.check()


@pytest.mark.parametrize("fmt", ["f16", "q8_0", "q4_0"])
@pytest.mark.parametrize("hd", [64, 128])
def test_read_cells(fmt, hd):
    """Cells in any order, one of them twice, against rows()."""
    rng = np.random.default_rng(3)
    kv = KvCache(2, 3, hd, 16 * 8, max_seqs=2, kv_format=fmt)
    n = 50
    cells = kv.append_batch(np.repeat([0, 1], [n, n]), np.tile(np.arange(n), 2))
    x = torch.from_numpy(rng.standard_normal((2, 2 * n, 3 * hd)).astype(np.float32)).cuda()
    kv.write(1, *cells, x[0], x[1])
    order = np.concatenate([rng.permutation(2 * n), [7, 7]])
    k, v = kv.read(1, cells[0][order], cells[1][order])
    for s in range(2):
        kr, vr = kv.rows(1, s, n)
        at = np.flatnonzero(order // n == s)
        assert torch.equal(k[at], kr[order[at] % n]) and torch.equal(v[at], vr[order[at] % n])
    k32, _ = kv.read(1, cells[0][order], cells[1][order], dtype=torch.float32)
    assert torch.equal(k32.half(), k)
    k0, v0 = kv.read(1, [], [])
    assert k0.shape == (0, 3 * hd)


def test_other_stream_and_two_caches():
    """Two caches on two streams at once, each with its own workspace."""
    rng = np.random.default_rng(13)
    ts, qs, outs = [], [], []
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for i in range(2):
        t = Twin(2, 128, 16 * 140, 8, max_seqs=2, max_batch=2048)
        with torch.cuda.stream(streams[i]):
            t.fill(0, 2000, rng)
            t.fill(1, 77 + i, rng)
        ts.append(t)
        qs.append(torch.from_numpy(rng.standard_normal((2, 8 * 128)).astype(np.float32)).cuda())
    torch.cuda.synchronize()
    for _ in range(5):
        for t, q, st in zip(ts, qs, streams):
            outs.append(t.kv.attend(0, q, [0, 1], [1999, t.kv.len(1) - 1], stream=st))
    torch.cuda.synchronize()
    for i, (t, q) in enumerate(zip(ts, qs)):
        ref = t.attend_ref(0, [0, 1], [1999, t.kv.len(1) - 1], q.cpu().numpy())
        for o in outs[i::2]:
            close(o, ref)


def test_refused_on_the_device():
    t = Twin(1, 64, 64, 4, max_seqs=2)
    rng = np.random.default_rng(0)
    t.fill(0, 20, rng)
    b = t.kv.seq_blocks(0)
    k, v = (torch.zeros((2, 64), device="cuda") for _ in range(2))
    with pytest.raises(KvError, match="named twice"):
        t.kv.write(0, [b[0], b[0]], [3, 3], k, v)
    with pytest.raises(KvError, match="out of range"):
        t.kv.read(0, [b[0], 99], [0, 0])
    with pytest.raises(KvError, match="out of range"):
        t.kv.read(3, [b[0]], [0])
    with pytest.raises(ValueError):
        t.kv.read(0, [b[0]], [0], k=torch.zeros((1, 64)), v=torch.zeros((1, 64)))
    big = torch.zeros(130, device="cuda")
    with pytest.raises(KvError, match="aligned"):
        t.kv.write(0, [b[0], b[1]], [0, 0], big[1:129].view(2, 64), v)
    t.check(0, 0)
    # a captured call would replay the staging and flags of the first one
    q = torch.zeros((1, 256), device="cuda")
    st = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    out = torch.empty((1, 256), device="cuda")
    with torch.cuda.graph(graph, stream=st):
        for call in (lambda: t.kv.attend(0, q, [0], [19], out=out, stream=st),
                     lambda: t.kv.write(0, b[:2], [0, 0], k, v, stream=st),
                     lambda: t.kv.read(0, b[:1], [0], k=k[:1], v=v[:1], stream=st),
                     lambda: t.kv.attend_shaped(0, q, [0], [19], window=4, out=out, stream=st)):
            with pytest.raises(KvError, match="captured"):
                call()
    t.kv.attend(0, q, [0], [19], out=out)
    t.kv.check()


def test_serving_run_of_everything_together():
    """Prefill, sharing, decode steps with fused appends, shaped attention on the
    same cache, truncation and regrowth, compaction, read-back: one run, each
    step against the restatement."""
    rng = np.random.default_rng(21)
    t = Twin(2, 128, 16 * 80, 8, layers=2, max_seqs=6)
    slopes = np.exp2(-np.arange(1, 9)).astype(np.float32)
    t.fill(0, 150, rng)
    for s in (1, 2, 3):
        t.kv.share(0, s, 140 + s)
        for layer in range(2):
            t.rows[(layer, s)] = list(t.rows[(layer, 0)][: 140 + s])
    t.fill(4, 37, rng)
    for step in range(12):
        seqs = np.array([0, 1, 2, 3, 4])
        pos = np.array([t.kv.len(s) for s in seqs])
        b, sl = t.kv.append_batch(seqs, pos)
        for layer in range(2):
            k, v = t.draw(5, rng)
            for i, s in enumerate(seqs):
                t.add(layer, int(s), k[i], v[i])
            q = rng.standard_normal((5, 8 * 128)).astype(np.float32)
            kd, vd, qd = (torch.from_numpy(x).cuda() for x in (k, v, q))
            close(t.kv.write_attend(layer, b, sl, kd, vd, qd, seqs, pos), t.attend_ref(layer, seqs, pos, q))
            first, end = np.array([0, 17, 140, 3, 20]), np.minimum(pos + 1, [150, 18, 200, 3, 40])
            out = t.kv.attend_shaped(layer, qd, seqs, pos, softcap=8.0, window=60, first=first, end=end,
                                     slopes=torch.from_numpy(slopes).cuda())
            for i, s in enumerate(seqs):
                K, V = t.values(layer, int(s))
                ref = A.attend(q[i].reshape(8, 128), K, V, int(pos[i]), 4, t.kv.default_scale, softcap=8.0, window=60,
                               first=first[i], end=end[i], slopes=slopes)
                close(out[i], ref.reshape(-1))
        if step == 5:
            t.kv.truncate(3, 33)
            for layer in range(2):
                del t.rows[(layer, 3)][33:]
            t.kv.truncate(0, 0)
            for layer in range(2):
                t.rows[(layer, 0)] = []
            assert t.kv.compact() > 0
            t.fill(0, 20, rng)
    for layer in range(2):
        for s in range(5):
            t.check(layer, s)
    t.kv.check()


def test_scheduler_over_a_4_bit_cache():
    """The native scheduler driver (admission, eviction, preemption, compaction,
    prefill and decode) moves 4-bit rows through the same calls: its last step's
    outputs are softmax attention over what the cache reads back."""
    from langtrain_studio_b200.sched import Scheduler

    hkv, hq, d, slots = 2, 8, 64, 6
    kv = KvCache(1, hkv, d, 16 * 60, n_heads=hq, max_seqs=slots, max_batch=512, kv_format="q4_0")
    sched = Scheduler(kv, slots)
    g = torch.Generator(device="cuda").manual_seed(5)
    kv_src = torch.randn((1024, hkv * d), generator=g, device="cuda", dtype=torch.float16)
    q_src = torch.randn((slots, hq * d), generator=g, device="cuda", dtype=torch.float16)
    out = torch.empty((slots, hq * d), device="cuda", dtype=torch.float16)
    rng = np.random.default_rng(6)
    decoded = 0
    for step in range(60):
        if step < 45:
            sched.submit(int(rng.integers(8, 250)), int(rng.integers(4, 40)))
        decoded += sched.step(kv_src, q_src, out)
    kv.check()
    assert decoded > 60 and sched.stats["finished"] > 0
    assert torch.isfinite(out.float()).all()


def test_llama_forward_over_a_4_bit_cache():
    """The Llama step runs on a 4-bit cache: the rows its first layer appends are
    the f16 cache's rows, quantised, and a prompt gives the same logits whether
    its tokens come together or one by one."""
    from langtrain_studio_b200 import llama as LL

    m = LL.Llama(2, 256, 4, 2, 64, 512, 500, max_batch=64)
    m.load(LL.random_weights(m, seed=3))
    toks = np.random.default_rng(0).integers(0, 500, 40)
    caches = {f: m.kv_cache(256, 2, kv_format=f) for f in ("f16", "q4_0")}
    logits = {f: m.forward(kv, toks, np.zeros(40), np.arange(40), [39]) for f, kv in caches.items()}
    for got, want in zip(caches["q4_0"].rows(0, 0, 40), caches["f16"].rows(0, 0, 40)):
        x = want.cpu().numpy().astype(np.float64).reshape(40, 2, 64)
        _, step = A.quant4(x)
        # half a step, a whole one past +7, and the step's own and the f16 row's rounding
        err = np.abs(got.cpu().numpy().reshape(x.shape) - x)
        assert (err <= np.repeat(np.abs(step), 32, -1) * (1 + 2 ** -6)).all()
    one = m.kv_cache(256, 2, kv_format="q4_0")
    for i, tok in enumerate(toks):
        lg = m.forward(one, [tok], [0], [i], [0])
    assert torch.isfinite(logits["q4_0"]).all()
    # attention differs by f32 rounding alone; the int8 activations may turn that
    # into single quantisation steps, a few per cent of the logits' spread
    assert (lg - logits["q4_0"]).abs().max() < 0.1 * logits["q4_0"].std()
    cos = torch.nn.functional.cosine_similarity(logits["q4_0"], logits["f16"]).item()
    assert cos > 0.8, cos


def test_peer_gather_single_rank():
    """The head-sharded gather over a 4-bit cache with one rank."""
    rng = np.random.default_rng(17)
    t = Twin(2, 128, 16 * 40, 8, max_seqs=3)
    lens = [40, 300, 17]
    for s, n in enumerate(lens):
        t.fill(s, n, rng)
    seqs, pos = np.arange(3), np.array(lens) - 1
    q = torch.from_numpy(rng.standard_normal((3, 8 * 128)).astype(np.float32)).cuda()
    want = t.kv.attend(0, q, seqs, pos)
    t.kv.peer_import([t.kv.peer_export(0, 1, max_tokens=8)])
    for _ in range(3):
        out = t.kv.attend_gather(0, q, seqs, pos, out_dtype=torch.float32)
        t.kv.check()
        assert torch.equal(out, want)
    t.kv.peer_close()
    t.kv.close()


@pytest.mark.parametrize("offset", [0, 1, 5, 15])
@pytest.mark.parametrize("hd", [64, 128])
def test_chunk_writes_at_any_offset(offset, hd):
    """Whole blocks, unaligned chunks, cells out of order and cells of several
    sequences in one write: the tile path and the row path meet in one call."""
    rng = np.random.default_rng(offset)
    t = Twin(3, hd, 16 * 40, max_seqs=3, max_batch=512)
    t.fill(0, offset, rng)
    t.fill(1, 3, rng)
    seqs = np.concatenate([np.zeros(70), np.ones(45), [2] * 16]).astype(np.int64)
    pos = np.concatenate([offset + np.arange(70), 3 + np.arange(45), np.arange(16)]).astype(np.int64)
    b, s = t.kv.append_batch(seqs, pos)
    k, v = t.draw(seqs.size, rng, np.float16)
    for i, q in enumerate(seqs):
        t.add(0, int(q), k[i], v[i])
    order = np.arange(seqs.size)
    order[100:] = rng.permutation(order[100:])
    t.kv.write(0, b[order], s[order], *(torch.from_numpy(np.ascontiguousarray(x[order])).cuda() for x in (k, v)))
    for q in range(3):
        t.check(0, q)
    kr, vr = t.kv.read(0, b[order], s[order])
    K = np.concatenate([t.values(0, q)[0][(offset, 3, 0)[q]:] for q in range(3)])
    assert np.array_equal(kr.cpu().numpy().astype(np.float64).reshape(K.shape), K[order])
    kr32, vr32 = t.kv.read(0, b, s, dtype=torch.float32)
    V = np.concatenate([t.values(0, q)[1][(offset, 3, 0)[q]:] for q in range(3)])
    assert np.array_equal(vr32.cpu().numpy().astype(np.float64).reshape(V.shape), V)


def test_rows_are_refused_in_a_capture():
    t = Twin(1, 64, 64, 4, max_seqs=2)
    t.fill(0, 20, np.random.default_rng(0))
    st = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    pad = torch.zeros(16, device="cuda")
    with torch.cuda.graph(graph, stream=st):
        pad.add_(1)
        with pytest.raises(KvError, match="captured"):
            t.kv.rows(0, 0, 20, stream=st)
    t.check(0, 0)


def test_offsets_past_32_bits():
    """A layer of more than 2^32 bytes: blocks behind them are written, read and attended."""
    blocks, hkv, hd, hq, n = 236000, 8, 128, 32, 100
    kv = KvCache(1, hkv, hd, 16 * blocks, n_heads=hq, max_seqs=2, max_batch=65536, max_blocks_per_seq=blocks,
                 kv_format="q4_0")
    assert kv.bytes() > 2 ** 32 + 2 ** 25
    used = 16 * (blocks - 8)
    for p0 in range(0, used, 65536):
        p = np.arange(p0, min(used, p0 + 65536), dtype=np.uint32)
        kv.append_batch(np.zeros(p.size, np.uint32), p)
    cells = kv.append_batch(np.ones(n, np.uint32), np.arange(n, dtype=np.uint32))
    assert int(min(cells[0])) * hkv * 18 * hd > 2 ** 32
    rng = np.random.default_rng(41)
    x = rng.standard_normal((2, n, hkv * hd)).astype(np.float32)
    kv.write(0, *cells, *(torch.from_numpy(a).cuda() for a in x))
    val = A.value4(*A.quant4(x.reshape(2, n, hkv, hd)))
    for got, want in zip(kv.read(0, *cells), val):
        assert np.array_equal(got.cpu().numpy().astype(np.float64), want.reshape(n, -1))
    for got, want in zip(kv.rows(0, 1, n), val):
        assert np.array_equal(got.cpu().numpy().astype(np.float64), want.reshape(n, -1))
    q = rng.standard_normal((n, hq * hd)).astype(np.float32)
    for first in (0, n - 1):  # a prefill chunk (through the prefix pass), a single token
        pos = np.arange(first, n)
        ref = np.stack([A.attend(q[i].reshape(hq, hd), *val, int(i), hq // hkv, kv.default_scale).reshape(-1) for i in pos])
        out = kv.attend(0, torch.from_numpy(q[first:]).cuda(), np.ones(pos.size), pos)
        shaped = kv.attend_shaped(0, torch.from_numpy(q[first:]).cuda(), np.ones(pos.size), pos, window=n)
        kv.check()
        for o in (out, shaped):
            np.testing.assert_allclose(o.cpu().numpy(), ref, rtol=1e-4, atol=2e-5)


@pytest.mark.parametrize("hd,hq,hkv", [(128, 32, 8), (64, 8, 2), (128, 16, 2), (64, 5, 1), (64, 16, 16)])
@pytest.mark.parametrize("dtype,out_dtype", [(torch.float32, torch.float32), (torch.float16, torch.float16),
                                             (torch.float16, torch.float32)])
def test_whole_chunks(hd, hq, hkv, dtype, out_dtype):
    """Calls of prefill chunks alone, which the pass attends whole: chunks from
    position 0, behind cached tokens, ends inside a block, tokens out of order
    and named twice, rows of a tile that no token has."""
    rng = np.random.default_rng(hd * hq + hkv)
    t = Twin(hkv, hd, 16 * 260, hq, max_seqs=8, max_batch=2048)
    for s, n in enumerate((8, 61, 127, 300, 1030, 97)):
        t.fill(s, n, rng)
    t.kv.share(4, 6, 600)  # two sequences on one prefix, each with its own chunk
    t.rows[(0, 6)] = list(t.rows[(0, 4)][:600])
    t.fill(6, 650, rng)
    chunks = [[(0, np.arange(8))], [(1, np.arange(61)), (2, np.arange(30, 127))],
              [(3, np.arange(300)), (4, np.arange(700, 1030)), (0, np.arange(8)), (6, np.arange(560, 650))],
              [(5, rng.permutation(97)), (4, np.r_[np.arange(1020, 1030), np.arange(1021, 1030)])]]
    for chunk in chunks:
        seqs = np.concatenate([np.full(p.size, s) for s, p in chunk])
        pos = np.concatenate([p for _, p in chunk])
        q = torch.from_numpy(rng.standard_normal((seqs.size, hq * hd)).astype(np.float32)).cuda().to(dtype)
        ref = t.attend_ref(0, seqs, pos, q.float().cpu().numpy())
        guard = torch.full((seqs.size + 2, hq * hd), 7.0, dtype=out_dtype, device="cuda")
        t.kv.attend(0, q, seqs, pos, out=guard[1:-1])
        t.kv.check()
        close(guard[1:-1], ref, out_dtype)
        assert (guard[0] == 7).all() and (guard[-1] == 7).all()


def test_whole_chunks_take_one_pass():
    """Of a call that the pass attends whole the tables are read by it alone:
    new blocks' entries are there, launches are its two, and what follows
    (a decode step, an append) finds everything as after any call."""
    rng = np.random.default_rng(3)
    t = Twin(8, 128, 16 * 300, 32, max_seqs=4, max_batch=1024)
    for s in range(4):
        t.fill(s, 200 + s, rng)
    for step in range(2):
        seqs, pos = np.repeat(np.arange(4), 80), np.concatenate([np.arange(80) + t.kv.len(s) for s in range(4)])
        cells = t.kv.append_batch(seqs, pos)
        k, v = t.draw(320, rng)
        q = rng.standard_normal((320, 32 * 128)).astype(np.float32)
        for s in range(4):
            t.add(0, s, k[seqs == s], v[seqs == s])
        c0, l0 = t.kv.cascade_launches(), t.kv.launch_count()
        out = t.kv.write_attend(0, *cells, *(torch.from_numpy(a).cuda() for a in (k, v, q)), seqs, pos)
        assert t.kv.cascade_launches() == c0 + 1
        assert t.kv.launch_count() - l0 <= 4  # plan, write, expansion, pass
        close(out, t.attend_ref(0, seqs, pos, q))
        s1, p1 = np.arange(4), np.array([t.kv.len(s) - 1 for s in range(4)])
        q1 = rng.standard_normal((4, 32 * 128)).astype(np.float32)
        close(t.kv.attend(0, torch.from_numpy(q1).cuda(), s1, p1), t.attend_ref(0, s1, p1, q1))
        for s in range(4):
            t.check(0, s)
    t.kv.check()


def test_a_cell_named_again_later_is_refused():
    t = Twin(1, 64, 64, 4, max_seqs=2)
    t.fill(0, 40, np.random.default_rng(0))
    b = t.kv.seq_blocks(0)
    k = torch.zeros((18, 64), device="cuda")
    for blocks, slots in (([b[0], b[1], b[0]], [3, 3, 3]), ([b[0], b[0], b[1], b[0]], [1, 2, 2, 2]),
                          ([b[0]] * 17 + [b[1]], list(range(16)) + [5, 0])):
        with pytest.raises(KvError, match="named twice"):
            t.kv.write(0, blocks, slots, k[:len(blocks)], k[:len(blocks)])
    t.check(0, 0)
    with pytest.raises(KvError, match="out of range"):
        t.kv.write(0, [b[0], b[0]], [3, 16], k[:2], k[:2])
    with pytest.raises(KvError, match="out of range"):
        t.kv.read(0, [b[0], -1], [3, 0])
    again = [b[1], b[0], b[1], b[0]], [3, 3, 4, 4]  # different slots of blocks that come again
    t.kv.write(0, *again, k[:4], k[:4])
    for got in t.kv.read(0, *again):
        assert not got.any()
    t.kv.check()


def test_short_runs_are_not_attended_whole():
    """Fewer than 8 tokens a sequence stay with the decode launch, whatever set_cascade says."""
    rng = np.random.default_rng(8)
    t = Twin(8, 128, 16 * 200, 32, max_seqs=20)
    for s in range(20):
        t.fill(s, 100 + s, rng)
    seqs = np.repeat(np.arange(20), 3)
    pos = np.array([t.kv.len(s) - 1 for s in seqs]) - np.tile([2, 1, 0], 20)
    q = rng.standard_normal((60, 32 * 128)).astype(np.float32)
    ref = t.attend_ref(0, seqs, pos, q)
    t.kv.set_cascade(4)
    c0 = t.kv.cascade_launches()
    close(t.kv.attend(0, torch.from_numpy(q).cuda(), seqs, pos), ref)
    assert t.kv.cascade_launches() == c0
    t.kv.check()


@pytest.mark.parametrize("gain,dtype", [(1e-6, torch.float32), (3e4, torch.float32), (1e6, torch.float32),
                                        (2e-6, torch.float16), (8e3, torch.float16)])
@pytest.mark.parametrize("hd,hq,hkv", [(128, 8, 2), (64, 9, 3)])
def test_chunks_and_prefixes_of_small_and_large_q(gain, dtype, hd, hq, hkv):
    """What test_attention_of_small_and_large_q asks of one token holds for prefill
    chunks and members of a shared prefix: they take another kernel."""
    rng = np.random.default_rng(51)
    t = Twin(hkv, hd, 16 * 120, hq, max_seqs=14)
    t.fill(0, 100, rng)
    for s in range(1, 12):
        t.kv.share(0, s, 70)
        t.rows[(0, s)] = list(t.rows[(0, 0)][:70])
        t.fill(s, 71 + 5 * (s % 4), rng)
    scale = float(np.float32(t.kv.default_scale / gain))
    slopes = np.exp2(-np.arange(1, hq + 1)).astype(np.float32)
    chunk = np.zeros(60, int), np.arange(40, 100)
    members = np.arange(1, 12), np.array([t.kv.len(s) - 1 for s in range(1, 12)])
    for (seqs, pos), shape in ((chunk, {}), (members, {}), (chunk, dict(softcap=5.0, window=40)),
                               (chunk, dict(slopes=slopes))):
        q = torch.from_numpy((rng.standard_normal((seqs.size, hq * hd)) * gain).astype(np.float32)).cuda().to(dtype)
        dev = {k: (torch.from_numpy(v).cuda() if k == "slopes" else v) for k, v in shape.items()}
        c0 = t.kv.cascade_launches()
        if shape:
            out = t.kv.attend_shaped(0, q, seqs, pos, scale=scale, **dev)
        else:
            out = t.kv.attend(0, q, seqs, pos, scale=scale)
        assert t.kv.cascade_launches() == c0 + 1
        ref = np.zeros((seqs.size, hq * hd))
        for i, (s, p) in enumerate(zip(seqs, pos)):
            ref[i] = A.attend(q[i].float().cpu().numpy().reshape(hq, hd), *t.values(0, int(s)), int(p), hq // hkv,
                              scale, **shape).reshape(-1)
        close(out, ref)
    t.kv.check()


def test_scheduler_outputs_over_a_4_bit_cache(oracle_mod):
    """Every step's outputs of the scheduler test above are attention over the rows
    that the policy has cached: the oracle, driven by the restated policy, holds the
    same rows after quantisation (its f16 values are the 4-bit ones exactly), and
    eviction, preemption and compaction leave every cell where it says."""
    import bench
    from langtrain_studio_b200.sched import Scheduler
    from oracle import churn

    hkv, hq, d, n_slots, pool = 2, 8, 64, 24, 96

    class Quantised:  # the driver's view of a cache, over the oracle
        def __init__(self):
            self.ok = oracle_mod.OracleKv(1, hkv * d, pool * 16, max_seqs=n_slots)
            for name in ("free_blocks", "truncate", "share", "seq_blocks", "refs"):
                setattr(self, name, getattr(self.ok, name))

        def append_batch(self, seqs, pos):
            rc, _, b, s = self.ok.append_batch(seqs, pos)
            assert rc == 0
            return b, s

        def write(self, layer, b, s, k, v):
            k, v = (A.value4(*A.quant4(x.reshape(-1, hkv, d))).astype(np.float16).reshape(-1, hkv * d) for x in (k, v))
            self.ok.write_batch(layer, b, s, k, v)

        def write_attend(self, layer, b, s, k, v, q, seqs, pos, out):
            self.write(layer, b, s, k, v)
            self.attended = np.zeros((len(seqs), hq * d))
            for i, (seq, p) in enumerate(zip(seqs, pos)):
                K, V = (r.view(np.float16).reshape(-1, hkv, d) for r in self.ok.rows(layer, int(seq), int(p) + 1))
                self.attended[i] = A.attend(q[i].reshape(hq, d), K, V, int(p), hq // hkv, kv.default_scale).reshape(-1)

        def compact(self):
            return len(self.ok.compact())

    kv = KvCache(1, hkv, d, 16 * pool, n_heads=hq, max_seqs=n_slots, max_batch=4096, max_blocks_per_seq=64,
                 kv_format="q4_0")
    sched, want = Scheduler(kv, n_slots), Quantised()
    g = torch.Generator(device="cuda").manual_seed(5)
    kv_src = torch.randn((4096, hkv * d), generator=g, device="cuda", dtype=torch.float16)
    q_src = torch.randn((n_slots, hq * d), generator=g, device="cuda", dtype=torch.float16)
    drv = churn.ChurnDriver(want, n_slots, kv_src.cpu().numpy(), q_src.cpu().numpy())
    arr = bench.Arrivals(1.5, 7, lo=8, hi=300, olo=4, ohi=40)
    for step in range(60):
        for p, o in arr.step():
            sched.submit(p, o)
            drv.submit(p, o)
        out = torch.full((n_slots, hq * d), float("nan"), device="cuda", dtype=torch.float16)
        nd = sched.step(kv_src, q_src, out)
        drv.step(np.zeros((n_slots, hq * d), np.float16))
        for s in range(n_slots):
            assert np.array_equal(kv.seq_blocks(s), want.seq_blocks(s)), (step, s)
        if nd:
            assert len(want.attended) == nd
            close(out[:nd], want.attended, torch.float16)
        assert out[nd:].isnan().all()  # rows behind the last token stay as they were
    st = sched.stats
    assert st["evicted"] > 0 and st["moved_blocks"] > 0 and st["decode_tokens"] > 60 and st["prefill_tokens"] > 0, st
    kc, vc, kd, vd = kv.pool_reference_layout(0)
    for codes, scales, ref in ((kc, kd, want.ok.pool()[0][0]), (vc, vd, want.ok.pool()[1][0])):
        got = A.value4(codes, scales.view(np.float16).astype(np.float64))
        assert np.array_equal(got.reshape(ref.shape), ref.view(np.float16).astype(np.float64))
    kv.check()
