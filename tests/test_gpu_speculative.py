"""The speculative-decoding operators on the GPU against plain 64-bit forms (tests/spec_cases.py): rotary positions, tree
attention, sampling, the accepted path's commit. Tolerances count roundings (the bounds are made with the references)."""
import ctypes

import numpy as np
import pytest

import spec_cases as S
from sardyne_amd import capi

pytestmark = pytest.mark.gpu

NAN16 = np.uint16(0x7E00)


def lib():
    capi.check(capi.lib().sdy_init())
    return capi.lib()


def up(a):
    return capi.DeviceBuffer.from_array(np.ascontiguousarray(a))


def as_kv(x, kv):
    """x as the cache holds it, and the values it then has."""
    h = x.astype(np.float16) if kv else x.astype(np.float32)
    return h, h.astype(np.float64)


# ----------------------------------------------------------------------------------- rotary

def run_rope(x, n_head, n_kv_head, hd, pos, slot, freq, mscale, n_rot, interleaved, kv, n_slot, qn=None, kn=None, eps=1e-6,
             in_place=False, pad=0, rows0=None, slot_at=0):
    """x [n][(n_head + 2 n_kv_head) hd + pad]: rows of stacked q|k|v -> q_out, k_rows, v_rows (as stored)."""
    n = x.shape[0]
    bx, bp, bf = up(x), up(pos.astype(np.int32)), up(freq)
    bs = up(np.concatenate([np.zeros(slot_at), slot]).astype(np.int32)) if slot is not None else None
    elt = np.float16 if kv else np.float32
    rows0 = np.full((2, n_kv_head, n_slot, hd), 7, elt) if rows0 is None else rows0
    bk, bv, bq = up(rows0[0]), up(rows0[1]), up(np.full((n, n_head * hd), 9, np.float32))
    norms = [up(w) if w is not None else None for w in (qn, kn)]
    q_dim, kv_dim = n_head * hd, n_kv_head * hd
    a = capi.SdyRopeAtArgs(q=bx.ptr, k=bx.ptr + 4 * q_dim, v=bx.ptr + 4 * (q_dim + kv_dim), q_stride=x.shape[1],
                           k_stride=x.shape[1], v_stride=x.shape[1], q_out=bx.ptr if in_place else bq.ptr,
                           q_out_stride=x.shape[1] if in_place else q_dim, k_rows=bk.ptr, v_rows=bv.ptr,
                           head_stride=n_slot * hd, kv_type=kv, n_slot=n_slot, pos=bp.ptr, slot=bs.ptr + 4 * slot_at if bs else None,
                           freq=bf.ptr, mscale=mscale, n_rot=n_rot, interleaved=interleaved,
                           q_norm=norms[0].ptr if norms[0] else None, k_norm=norms[1].ptr if norms[1] else None, eps=eps,
                           n_tok=n, n_head=n_head, n_kv_head=n_kv_head, hd=hd)
    capi.check(lib().sdy_qk_rope_at(ctypes.byref(a), None))
    q = bx.to_array(np.float32, x.shape)[:, :q_dim] if in_place else bq.to_array(np.float32, (n, q_dim))
    return (q.reshape(n, n_head, hd), bk.to_array(elt, rows0.shape[1:]), bv.to_array(elt, rows0.shape[1:]))


def rope_freq(n_rot, kind=None):
    f, m = np.empty(max(n_rot // 2, 1)), ctypes.c_float()
    sc = capi.SdyRopeScaling(kind=kind or 0, factor=8.0, orig_ctx=4096, beta_fast=32.0, beta_slow=1.0, low_freq=1.0,
                             high_freq=4.0)
    capi.check(capi.lib().sdy_rope_freqs(f.ctypes.data, ctypes.byref(m), n_rot, 1e6, ctypes.byref(sc)))
    return f, m.value


@pytest.mark.parametrize("n,nh,nkv,hd,n_rot,kind,past", [
    (1, 1, 1, 64, 64, 0, 0), (1, 16, 2, 128, 128, 0, 511), (5, 4, 4, 64, 32, 1, 70_000), (61, 32, 4, 128, 128, 2, 9000),
    (300, 8, 8, 128, 64, 3, 1_000_000), (7, 7, 1, 256, 256, 2, 3), (3, 2, 1, 122, 122, 3, 2_000_000_000), (9, 3, 3, 80, 20, 0, 17),
    (4, 2, 2, 128, 0, 0, 5), (33, 6, 2, 96, 90, 1, 12345), (2, 1, 1, 2, 2, 0, 1), (3, 2, 1, 512, 512, 0, 77),
    (11, 14, 2, 64, 58, 2, 400), (6, 5, 5, 32, 32, 3, 99), (13, 40, 8, 128, 8, 0, 31)])
@pytest.mark.parametrize("interleaved", [0, 1])
@pytest.mark.parametrize("norm", [False, True], ids=["plain", "norm"])
@pytest.mark.parametrize("kv", [0, 1], ids=["f32", "f16"])
def test_rope_at(n, nh, nkv, hd, n_rot, kind, past, interleaved, norm, kv):
    rng = np.random.default_rng(n * 1000 + hd + n_rot)
    pad = int(rng.integers(0, 4)) * (1 if n % 2 else 4)
    x = rng.standard_normal((n, (nh + 2 * nkv) * hd + pad)).astype(np.float32)
    pos = past + np.array([max(0, int(d)) for d in rng.integers(0, n + 1, n)])
    n_slot = n + 3
    slot = rng.permutation(n_slot)[:n]
    slot[n // 2] = [-1, n_slot, -2**31][n % 3]  # no row for this one
    freq, mscale = rope_freq(n_rot, kind)
    qn, kn = ((1 + 0.2 * rng.standard_normal(hd)).astype(np.float32) for _ in range(2)) if norm else (None, None)
    q, k, v = run_rope(x, nh, nkv, hd, pos, slot, freq, mscale, n_rot, interleaved, kv, n_slot, qn, kn)
    parts = np.split(x[:, :(nh + 2 * nkv) * hd].reshape(n, nh + 2 * nkv, hd), [nh, nh + nkv], axis=1)
    eq, tq = S.rope(parts[0], pos, freq[:n_rot // 2], mscale, n_rot, interleaved, qn, 1e-6)
    assert (np.abs(q - eq) <= tq + 1e-30).all()
    ek, tk = S.rope(parts[1], pos, freq[:n_rot // 2], mscale, n_rot, interleaved, kn, 1e-6)
    want_k, want_v = np.full((nkv, n_slot, hd), 7.0), np.full((nkv, n_slot, hd), 7.0)
    tol = np.zeros((nkv, n_slot, hd))
    for t in range(n):
        if 0 <= slot[t] < n_slot:
            want_k[:, slot[t]], tol[:, slot[t]] = ek[t], tk[t]
            want_v[:, slot[t]] = as_kv(parts[2][t], kv)[1]
    if kv:
        tol = tol + np.abs(want_k) * S.U16 * (1 + 2.0 ** -10) + 2.0 ** -25
    assert (np.abs(k.astype(np.float64) - want_k) <= tol + 1e-30).all()
    assert np.array_equal(v.astype(np.float64), want_v)


@pytest.mark.parametrize("interleaved", [0, 1])
@pytest.mark.parametrize("kv", [0, 1], ids=["f32", "f16"])
def test_rope_at_is_the_consecutive_form(interleaved, kv):
    """Whole unscaled heads at pos0 + t: the values of sdy_qk_rope_kv with the host's tables, bit for bit."""
    n, nh, nkv, hd, pos0, max_seq = 40, 4, 2, 128, 700, 800
    rng = np.random.default_rng(5)
    x = rng.standard_normal((n, (nh + 2 * nkv) * hd)).astype(np.float32)
    cos, sin = (np.empty((max_seq, hd // 2), np.float32) for _ in range(2))
    capi.lib().op_rope_table(cos.ctypes.data, sin.ctypes.data, max_seq, hd, 1e6)
    bx, bc, bn = up(x), up(cos), up(sin)
    elt = np.float16 if kv else np.float32
    zero = np.full((2, nkv, max_seq, hd), 7, elt)
    bk, bv = up(zero[0]), up(zero[1])
    w = x.shape[1]
    capi.check(lib().sdy_qk_rope_kv_strided(bx.ptr, bx.ptr + 4 * nh * hd, bx.ptr + 4 * (nh + nkv) * hd, w, w, w, None, None,
                                            0.0, bc.ptr, bn.ptr, pos0, n, nh, nkv, hd, interleaved, bk.ptr, bv.ptr, kv,
                                            max_seq * hd, None))
    want_q = bx.to_array(np.float32, x.shape)[:, :nh * hd].reshape(n, nh, hd)
    freq, mscale = rope_freq(hd)
    for in_place in (False, True):
        q, k, v = run_rope(x, nh, nkv, hd, pos0 + np.arange(n), None, freq, mscale, hd, interleaved, kv, max_seq,
                           in_place=in_place)
        assert np.array_equal(q.view(np.uint32), want_q.view(np.uint32))
        assert k.tobytes() == bk.to_array(elt, zero.shape[1:]).tobytes()
        assert v.tobytes() == bv.to_array(elt, zero.shape[1:]).tobytes()


@pytest.mark.parametrize("n,at", [(600, 0), (601, 0), (603, 1), (5, 0), (2, 3), (2050, 2), (4103, 0)])
def test_rope_at_one_slot_for_several_tokens(n, at):
    """The last of them stays, wherever the others ran, and wherever the slots lie."""
    nkv, hd = 2, 64
    rng = np.random.default_rng(8)
    x = rng.standard_normal((n, 3 * nkv * hd)).astype(np.float32)
    slot = rng.integers(0, 7, n)
    freq, mscale = rope_freq(hd)
    _, _, v = run_rope(x, nkv, nkv, hd, np.arange(n), slot, freq, mscale, hd, 0, 0, 8, slot_at=at)
    want = np.full((nkv, 8, hd), 7, np.float32)
    for t in range(n):
        want[:, slot[t]] = x[t, 2 * nkv * hd:].reshape(nkv, hd)
    assert np.array_equal(v, want)


def test_rope_at_negative_positions_turn_back():
    hd, n = 128, 6
    x = np.random.default_rng(2).standard_normal((n, 3 * hd)).astype(np.float32)
    pos = np.array([-1, -500, -(2**31), 2**31 - 1, 0, 3])
    freq, mscale = rope_freq(hd)
    q, _, _ = run_rope(x, 1, 1, hd, pos, np.arange(n), freq, mscale, hd, 0, 0, n)
    want, tol = S.rope(x[:, None, :hd], pos, freq, mscale, hd, 0)
    # the angle itself is a product in 64 bits: half a step of 2^31 radians is 2^-23
    tol = tol + np.abs(x[:, None, :hd]).max() * 2 * np.abs(pos)[:, None, None] * 2.0 ** -53
    assert (np.abs(q - want) <= tol).all()


@pytest.mark.parametrize("part", ["q", "k"])
def test_rope_at_queries_or_keys_alone(part):
    n, hd = 5, 64
    rng = np.random.default_rng(4)
    x = rng.standard_normal((n, 3 * hd)).astype(np.float32)
    freq, _ = rope_freq(hd)
    bx, bp, bf = up(x), up(np.arange(n, dtype=np.int32)), up(freq)
    bq, bk, bv = (up(np.full((n, hd), 7, np.float32)) for _ in range(3))
    a = capi.SdyRopeAtArgs(q_stride=3 * hd, k_stride=3 * hd, v_stride=3 * hd, q_out_stride=hd, head_stride=n * hd, n_slot=n,
                           pos=bp.ptr, freq=bf.ptr, mscale=1.0, n_rot=hd, n_tok=n, n_head=1, n_kv_head=1, hd=hd)
    if part == "q":
        a.q, a.q_out = bx.ptr, bq.ptr
    else:
        a.k, a.v, a.k_rows, a.v_rows = bx.ptr + 4 * hd, bx.ptr + 8 * hd, bk.ptr, bv.ptr
    capi.check(lib().sdy_qk_rope_at(ctypes.byref(a), None))
    got = [b.to_array(np.float32, (n, hd)) for b in (bq, bk, bv)]
    for i, name in enumerate("qkv"):
        if (name == "q") != (part == "q"):
            assert (got[i] == 7).all()
        elif name == "v":
            assert np.array_equal(got[i], x[:, 2 * hd:])
        else:
            want, tol = S.rope(x[:, None, i * hd:(i + 1) * hd], np.arange(n), freq, 1.0, hd, 0)
            assert (np.abs(got[i] - want[:, 0]) <= tol[:, 0]).all()


# ----------------------------------------------------------------------------------- tree attention

class Tree:
    """Inputs of one tree attention on the GPU. Cache rows past the bound's last used one, unused nodes' rows and queries
    hold NaN."""

    def __init__(self, n, past, nh, nkv, hd, kv, seed, unused=0, max_past=None, q_scale=1.0, parent=None, spike=None):
        rng = np.random.default_rng(seed)
        self.n, self.nh, self.nkv, self.hd, self.kv, self.past = n, nh, nkv, hd, kv, past
        self.max_past = past + 37 if max_past is None else max_past
        rows = max(self.max_past, 1)
        self.parent = S.random_tree(n, rng, unused=unused, roots=0.1) if parent is None else np.array(parent, np.int32)
        q = (q_scale * rng.standard_normal((n, nh, hd))).astype(np.float32)
        kv_of = lambda *s: rng.standard_normal(s).astype(np.float16 if kv else np.float32)  # noqa: E731
        self.cache, self.draft = [kv_of(nkv, rows, hd), kv_of(nkv, rows, hd)], [kv_of(nkv, n, hd), kv_of(nkv, n, hd)]
        if spike:
            spike(q, self.cache, self.draft)
        for c in self.cache:
            c[:, past:] = np.nan
        for d in self.draft:
            d[:, self.parent < -1] = np.nan
        q[self.parent < -1] = np.nan
        self.q = q
        self.want, self.tol = S.tree_attention(q, *self.cache, *self.draft, past, self.parent)
        self.b = [up(x) for x in (q, *self.cache, *self.draft, self.parent, np.array([past], np.int32))]
        self.out = up(np.full((n, nh, hd), 7, np.float32))
        floats = lib().sdy_attn_tree_floats(n, nh, nkv, hd, self.max_past)
        self.part = up(np.full(floats + 64, np.nan, np.float32))
        p = [b.ptr for b in self.b]
        self.args = capi.SdyAttnTreeArgs(q=p[0], q_stride=nh * hd, k_cache=p[1], v_cache=p[2], head_stride=rows * hd,
                                         k_draft=p[3], v_draft=p[4], draft_stride=n * hd, kv_type=kv, parent=p[5],
                                         n_past=p[6], max_past=self.max_past, n_tok=n, n_head=nh, n_kv_head=nkv, hd=hd,
                                         out=self.out.ptr, out_stride=nh * hd, part=self.part.ptr)

    def run(self, stream=None):
        capi.check(lib().sdy_attn_tree(ctypes.byref(self.args), stream))
        return self

    def got(self, stream=None):
        return self.out.to_array(np.float32, (self.n, self.nh, self.hd), stream)

    def check(self, got=None):
        got = self.got() if got is None else got
        used = self.parent >= -1
        assert (got[~used] == 7).all()
        assert np.isfinite(got[used]).all()
        off = np.abs(got - self.want)[used] / self.tol[used]
        assert off.max(initial=0) <= 1, off.max()
        return got


@pytest.mark.parametrize("n,past,nh,nkv,hd", [
    (1, 0, 1, 1, 64), (1, 1, 2, 1, 128), (1, 700, 16, 2, 128), (2, 31, 4, 4, 64), (3, 32, 8, 1, 128), (5, 33, 7, 1, 64),
    (4, 63, 8, 2, 128), (8, 64, 4, 1, 256), (9, 65, 16, 2, 128), (16, 127, 8, 1, 128), (17, 128, 32, 4, 64),
    (31, 0, 4, 2, 128), (33, 129, 14, 2, 64), (61, 500, 8, 1, 128), (64, 1023, 16, 2, 128), (65, 1024, 4, 1, 64),
    (100, 40, 16, 1, 128), (128, 301, 4, 2, 256), (255, 77, 8, 2, 64), (256, 256, 4, 4, 128), (24, 5000, 8, 1, 128),
    (2, 24700, 8, 8, 128), (3, 6000, 16, 16, 64), (50, 3000, 4, 1, 64)])
@pytest.mark.parametrize("kv", [0, 1], ids=["f32", "f16"])
def test_attn_tree(n, past, nh, nkv, hd, kv):
    Tree(n, past, nh, nkv, hd, kv, n + past, unused=3 if n > 8 else 0).run().check()


@pytest.mark.parametrize("past,max_past", [(0, 0), (0, 5000), (3, 5000), (5000, 5000), (4999, 20000), (511, 1 << 20)])
def test_attn_tree_bound_and_position(past, max_past):
    """The bound sets the split of the work, not the result; the caches need not have rows up to it... only up to n_past."""
    if max_past > 20000:
        t = Tree(9, past, 4, 1, 64, 0, 3, max_past=past)
        t.args.max_past = max_past
        floats = lib().sdy_attn_tree_floats(9, 4, 1, 64, max_past)
        t.part = up(np.full(floats, np.nan, np.float32))
        t.args.part = t.part.ptr
        t.run().check()
    else:
        Tree(9, past, 4, 2, 128, 0, 3, max_past=max_past).run().check()


@pytest.mark.parametrize("kind", ["chain", "star", "roots", "bad_parents", "all_unused", "hole"])
def test_attn_tree_shapes_of_trees(kind):
    n = 70
    parent = {"chain": list(range(-1, n - 1)), "star": [-1] + [0] * (n - 1), "roots": [-1] * n,
              "bad_parents": [5, 1, 1, 100, -1] + [2**31 - 1, -1] * ((n - 5) // 2) + [n - 1], "all_unused": [-2] * n,
              "hole": [-1, 0, -2, 2, 3] + [-(2**31)] * 5 + [9] * (n - 10)}[kind]
    for kv in (0, 1):
        Tree(n, 90, 8, 2, 64, kv, 1, parent=parent).run().check()


@pytest.mark.parametrize("past", [-1, 91, 2**31 - 1, -(2**31)])
def test_attn_tree_position_outside_leaves_out(past):
    t = Tree(20, 90, 8, 2, 64, 0, 1, max_past=90)
    b = up(np.array([past], np.int32))
    t.args.n_past = b.ptr
    assert (t.run().got() == 7).all()


@pytest.mark.parametrize("kv", [0, 1], ids=["f32", "f16"])
@pytest.mark.parametrize("what", ["peaks", "large", "tiny", "vanishing", "mixed_rows", "equal"])
def test_attn_tree_values(what, kv):
    def spike(q, cache, draft):
        if what == "peaks":  # weights that leave one position
            cache[0][:, ::7] *= 30
        if what == "large":
            q *= 100
            cache[1] *= 1000
        if what == "tiny":
            q *= 1e-6
            for x in cache + draft:
                x *= 1e-3
        if what == "vanishing":  # scores of 0 from K and q that are not, and from a q that is
            q[:] *= np.float32(1e-38)
            q[::3] = 0
            for x in cache[:1] + draft[:1]:
                x *= x.dtype.type(1e-35 if x.dtype == np.float32 else 1e-7)
        if what == "mixed_rows":  # rows of very different sizes, and dims within a row
            q *= np.exp2(np.arange(-10, 10))[None, None, np.arange(q.shape[2]) % 20].astype(q.dtype) / 8
            cache[0][:, ::3] /= 256
            cache[1][:, ::5] *= 512
            draft[1][:, ::2] /= 512
        if what == "equal":
            for x in cache + draft:
                x[:] = 1
    Tree(37, 333, 8, 2, 128, kv, 6, spike=spike).run().check()


@pytest.mark.parametrize("kv", [0, 1], ids=["f32", "f16"])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("n,nh", [(12, 8), (90, 8)])
def test_attn_tree_bad_drafted_rows(bad, kv, n, nh):
    """A drafted row with a value that is no number: NaN for the nodes that see it, nothing for the others."""
    t = Tree(n, 100, nh, 2, 64, kv, 21)
    node = n // 3
    for side in (0, 1):
        rows = t.draft[side].copy()
        rows[1, node, 5] = bad
        b = up(rows)
        args = type(t.args).from_buffer_copy(t.args)
        setattr(args, ("k_draft", "v_draft")[side], b.ptr)
        capi.check(lib().sdy_attn_tree(ctypes.byref(args), None))
        got = t.got()
        sees = S.ancestors(t.parent)[:, node]
        assert sees.any() and not sees.all()
        assert np.isnan(got[sees][:, nh // 2:]).all()
        t.want[sees, nh // 2:] = got[sees, nh // 2:] = 0
        t.check(got)


def test_attn_tree_strided_rows():
    t = Tree(21, 150, 4, 2, 64, 0, 2)
    wide_q, wide_o = np.full((21, 4 * 64 + 12), np.nan, np.float32), np.full((21, 4 * 64 + 20), 7, np.float32)
    wide_q[:, :256] = t.q.reshape(21, 256)
    bq, bo = up(wide_q), up(wide_o)
    t.args.q, t.args.q_stride, t.args.out, t.args.out_stride = bq.ptr, 268, bo.ptr, 276
    got = t.run() and bo.to_array(np.float32, wide_o.shape)
    assert (got[:, 256:] == 7).all()
    t.check(got[:, :256].reshape(21, 4, 64))


def test_attn_tree_same_bits_every_call_and_in_a_graph():
    """Eagerly, again, and replayed for several positions and trees while other calls run between, two graphs in turn on
    one scratch: one result per input."""
    L = lib()
    st = ctypes.c_void_p()
    capi.check(L.sdy_stream_new(ctypes.byref(st)))
    t = Tree(40, 900, 8, 2, 128, 0, 9, max_past=1500)
    first = t.run().check()
    assert np.array_equal(t.run().got().view(np.uint32), first.view(np.uint32))
    other = Tree(7, 1200, 8, 2, 128, 0, 10, max_past=1500)
    big = max(t.part.nbytes, other.part.nbytes)
    shared = capi.DeviceBuffer(big)
    graphs = []
    for x in (t, other):
        x.args.part = shared.ptr
        capi.check(L.sdy_sync(None))
        capi.check(L.sdy_graph_begin(st))
        x.run(st)
        g = ctypes.c_void_p()
        capi.check(L.sdy_graph_end(st, ctypes.byref(g)))
        graphs.append(g)
    want = [first, Tree(7, 1200, 8, 2, 128, 0, 10, max_past=1500).run().check()]
    for k in range(6):
        for x, g, w in zip((t, other), graphs, want):
            capi.check(L.sdy_memset(x.out.ptr, 0, x.out.nbytes, st))
            capi.check(L.sdy_graph_launch(g, st))
            assert np.array_equal(x.got(st).view(np.uint32), w.view(np.uint32)), k
        Tree(3, 50 * k, 4, 2, 64, 1, k).run().check()
    # a replay at another position
    t2 = Tree(40, 900, 8, 2, 128, 0, 9, max_past=1500)
    short = np.array([123], np.int32)
    capi.check(L.sdy_h2d(t.b[6].ptr, short.ctypes.data, 4, st))
    capi.check(L.sdy_graph_launch(graphs[0], st))
    t2.want, t2.tol = S.tree_attention(t2.q, *t2.cache, *t2.draft, 123, t2.parent)
    t2.check(t.got(st))
    for g in graphs:
        capi.check(L.sdy_graph_free(g))
    capi.check(L.sdy_stream_free(st))


# ----------------------------------------------------------------------------------- sampling

def run_sample(x, temp=None, top_k=None, top_p=None, min_p=None, u=None, pad=0, prob=True, offset=0):
    n, v = x.shape
    wide = np.full((n, v + pad), np.inf, np.float32)  # what stands between the rows is never looked at
    wide[:, :v] = x
    flat = np.full(wide.size + offset, np.inf, np.float32)
    flat[offset:] = wide.reshape(-1)
    f = lambda a, t: None if a is None else up(np.broadcast_to(np.asarray(a, t), n))  # noqa: E731
    b = [up(flat), f(temp, np.float32), f(top_k, np.int32), f(top_p, np.float32), f(min_p, np.float32),
         f(u, np.float32)]
    tok, pr = up(np.full(n + 1, 77, np.int32)), up(np.full(n + 1, 77, np.float32))
    ws = capi.DeviceBuffer(lib().sdy_sample_ws_bytes(n, v))
    capi.check(lib().sdy_memset(ws.ptr, 0xA5, ws.nbytes, None))
    p = [x.ptr if x else None for x in b]
    a = capi.SdySampleArgs(logits=p[0] + 4 * offset, stride=v + pad, n_rows=n, n_vocab=v, temp=p[1], top_k=p[2], top_p=p[3],
                           min_p=p[4], u=p[5], token=tok.ptr, prob=pr.ptr if prob else None, ws=ws.ptr)
    capi.check(lib().sdy_sample(ctypes.byref(a), None))
    t, q = tok.to_array(np.int32, n + 1), pr.to_array(np.float32, n + 1)
    assert t[n] == 77 and q[n] == 77
    return t[:n], q[:n]


def check_sample(x, temp=None, top_k=None, top_p=None, min_p=None, u=None, **kw):
    got, prob = run_sample(x, temp, top_k, top_p, min_p, u, **kw)
    row = lambda a, r, d: d if a is None else np.broadcast_to(np.asarray(a, np.float32), len(x))[r]  # noqa: E731
    for r in range(len(x)):
        k = 0 if top_k is None else int(np.broadcast_to(np.asarray(top_k, np.int64), len(x))[r])
        want, p = S.sample(x[r], row(temp, r, np.float32(1)), k, row(top_p, r, np.float32(1)), row(min_p, r, np.float32(0)),
                           row(u, r, None))
        assert got[r] == want, (r, got[r], want)
        # rounded once, from sums of whole multiples of at most 2^-40 of the greatest weight
        assert abs(prob[r] - p) <= S.U32 * p * 1.01 + 1e-30 + 2.0 ** -39, (r, prob[r], p)


@pytest.mark.parametrize("n,v", [(1, 1), (3, 2), (5, 17), (4, 63), (3, 64), (7, 257), (2, 1023), (3, 1025), (4, 2560), (4, 2561), (40, 4099),
                                 (9, 32000), (300, 1500), (2, 151936), (70, 5003), (1, 262147)])
@pytest.mark.parametrize("kind", ["float", "coarse", "masked", "flat", "steep"])
def test_sample(n, v, kind):
    rng = np.random.default_rng(v + n)
    x = (2 * rng.standard_normal((n, v)) + 1.3 * rng.exponential(size=(n, v))).astype(np.float32)
    if kind == "coarse":
        x = np.round(x * 4) / 4
    if kind == "masked":
        x[rng.random((n, v)) < 0.9] = [-np.inf, np.finfo(np.float32).min][v % 2]
    if kind == "flat":
        x = (x * 1e-3).astype(np.float32)
    if kind == "steep":
        x *= 20
    check_sample(x, rng.choice([0, 0.3, 0.7, 1.0, 1.5], n), rng.choice([0, 1, 2, 20, 50, 400, v, v + 1, -1], n),
                 rng.choice([0, 0.1, 0.5, 0.8, 0.95, 0.999, 1, 2], n), rng.choice([0, 0, 0.01, 0.05, 0.5, 1, 1.5], n),
                 rng.random(n), pad=int(rng.integers(0, 5)), offset=int(rng.integers(0, 4)))


@pytest.mark.parametrize("top_k", [1000, 4095, 4096, 4097, 5000, 30000, 79999, 80000])
def test_sample_many_kept(top_k):
    rng = np.random.default_rng(top_k)
    x = (2 * rng.standard_normal((4, 80000))).astype(np.float32)
    x[1] = np.round(x[1] * 2) / 2  # thousands of ties at every border
    x[2] = 0.25
    x[3] = np.round(x[3]) * 50
    check_sample(x, [1.2, 0.9, 1.0, 3.0], top_k, [1.0, 0.7, 0.6, 0.9], 0.0, rng.random(4))
    check_sample(x, [1.2, 0.9, 1.0, 3.0], top_k, 1.0, [0.0, 0.001, 0.0, 0.0], rng.random(4))
    check_sample(x, 2.0, None, [0.3, 0.99, 0.9999, 0.5], None, rng.random(4))


def test_sample_defaults_and_no_prob():
    rng = np.random.default_rng(0)
    x = rng.standard_normal((6, 999)).astype(np.float32)
    u = rng.random(6).astype(np.float32)
    check_sample(x, u=u)
    got, prob = run_sample(x, u=u, prob=False)
    assert (prob == 77).all() and np.array_equal(got, run_sample(x, u=u)[0])


@pytest.mark.parametrize("v", [5, 3001])
def test_sample_special_logits(v):
    nan, inf, low = np.nan, np.inf, np.finfo(np.float32).min
    rng = np.random.default_rng(1)
    x = rng.standard_normal((12, v)).astype(np.float32)
    x[0] = -inf
    x[1] = nan
    x[2] = low
    x[3, ::2] = nan
    x[4, 3] = inf
    x[5, 1] = x[5, 4] = inf
    x[6, :] = -inf
    x[6, 2] = low
    x[7] = -0.0
    x[7, 3] = 0.0
    x[8] = -inf
    x[8, 1:3] = nan
    x[9] = 3.0e38
    x[9, 1] = -3.0e38
    x[10] = 1e-45
    x[11] = np.arange(v)[::-1] * np.float32(1e-3)
    for temp in (0.0, 1e-30, 0.5, 1.0, 1e30, inf, nan, -1.0):
        for top_p, top_k, min_p in ((1.0, 0, 0.0), (0.9, 0, 0.0), (1.0, 2, 0.0), (0.5, 3, 0.1)):
            for u in (0.0, 0.37, 0.9999999):
                check_sample(x, temp, top_k, top_p, min_p, u)
    for u in (-1.0, -inf, nan):
        assert np.array_equal(run_sample(x, u=u)[0], run_sample(x, u=0.0)[0])
    for u in (1.0, 2.0, inf):
        assert np.array_equal(run_sample(x, u=u)[0], run_sample(x, u=np.float32(1) - np.float32(2.0 ** -24))[0])


@pytest.mark.parametrize("v", [2561, 4099, 40003])
def test_sample_special_long_rows(v):
    """As above in rows that are cut into pieces: what decides is where the bins of distance from the greatest logit end."""
    nan, inf, big = np.nan, np.inf, np.float32(3e38)
    rng = np.random.default_rng(v)
    x = rng.standard_normal((10, v)).astype(np.float32)
    x[1] = -inf
    x[1, 7::9] = nan
    x[2, 5::1000] = inf
    x[3] *= big / 8
    x[4] = np.where(rng.random(v) < 0.5, big, -big)
    x[5, :] = -inf
    x[5, v - 1] = np.finfo(np.float32).min
    x[6] = -0.0
    x[6, 3] = 0.0
    x[7] = 1e-45 * (np.arange(v) % 5)
    x[8, rng.random(v) < 0.5] = nan
    x[9] = inf
    for temp in (0.0, 1e-45, 1.0, 1e19, 1e38, inf, nan):
        for top_p, top_k, min_p in ((1.0, 0, 0.0), (0.9, 0, 0.0), (1.0, 0, 1.0), (1.0, 0, 0.03), (0.6, 0, 0.5), (1.0, 2000, 0.03),
                                    (0.5, 300, 0.0), (0.0, 0, 2.0)):
            check_sample(x, temp, top_k, top_p, min_p, rng.random(10))
    u = rng.random(10)  # no numbers: as if not given
    assert np.array_equal(run_sample(x, 2.0, 0, nan, nan, u)[0], run_sample(x, 2.0, u=u)[0])


def test_sample_follows_the_probabilities():
    """Every token of a small row is taken by just the u of its share."""
    x = np.log(np.array([[0.1, 0.0, 0.35, 0.05, 0.5]], np.float32) + 1e-45).astype(np.float32)
    u = (np.arange(2000) + 0.5) / 2000
    got, _ = run_sample(np.repeat(x, 2000, 0), u=u.astype(np.float32))
    assert np.array_equal(np.bincount(got, minlength=5), [200, 0, 700, 100, 1000])
    got, prob = run_sample(np.repeat(x, 2000, 0), top_p=0.8, u=u.astype(np.float32))
    assert set(got) == {2, 4} and abs(prob[got == 4][0] - 0.5 / 0.85) < 1e-6


# ----------------------------------------------------------------------------------- the commit

def run_commit(token, parent, sampled, past, draft, cache, kv, stream=None):
    n = len(token)
    nl, nkv, max_seq, hd = cache.shape[1:]
    b = [up(np.asarray(x, np.int32)) for x in (token, parent, sampled, [past])]
    bd, bc = [up(d) for d in draft], [up(c) for c in cache]
    o = [up(np.full(k, 77, np.int32)) for k in (n + 1, 2, 3)]
    a = capi.SdyTreeCommitArgs(token=b[0].ptr, parent=b[1].ptr, sampled=b[2].ptr, n_tok=n, n_past=b[3].ptr,
                               k_draft=bd[0].ptr, v_draft=bd[1].ptr, draft_stride=draft.shape[3] * hd,
                               draft_layer_stride=nkv * draft.shape[3] * hd, k_cache=bc[0].ptr, v_cache=bc[1].ptr,
                               head_stride=max_seq * hd, layer_stride=nkv * max_seq * hd, kv_type=kv, max_seq=max_seq,
                               n_layer=nl, n_kv_head=nkv, hd=hd, path=o[0].ptr, n_acc=o[1].ptr, step=o[2].ptr)
    capi.check(lib().sdy_tree_commit(ctypes.byref(a), stream))
    path, acc, step = (x.to_array(np.int32, k, stream) for x, k in zip(o, (n + 1, 2, 3)))
    assert path[n] == 77 and acc[1] == 77 and step[2] == 77
    return path[:n], int(acc[0]), step[:2], np.stack([x.to_array(cache.dtype, cache.shape[1:], stream) for x in bc])


@pytest.mark.parametrize("n,nl,nkv,hd,max_seq,past", [
    (1, 1, 1, 64, 1, 0), (8, 3, 2, 128, 40, 7), (61, 5, 4, 128, 80, 19), (256, 2, 1, 64, 300, 44), (30, 1, 8, 256, 33, 31),
    (12, 2, 3, 7, 50, 20), (9, 4, 1, 66, 12, 11), (5, 2, 2, 128, 9, 9), (5, 2, 2, 128, 9, -1), (64, 2, 2, 20, 70, 3)])
@pytest.mark.parametrize("kv", [0, 1], ids=["f32", "f16"])
@pytest.mark.parametrize("agree", [0.0, 0.85, 1.0])
def test_tree_commit(n, nl, nkv, hd, max_seq, past, kv, agree):
    rng = np.random.default_rng(n + hd)
    elt = np.float16 if kv else np.float32
    parent = S.random_tree(n, rng, back=3, unused=2 if n > 8 else 0)
    token = rng.integers(0, 1000, n)
    sampled = rng.integers(1000, 2000, n)
    for t in range(1, n):
        if parent[t] >= 0 and rng.random() < agree:
            sampled[parent[t]] = token[t]
    if n > 4:  # twins: the lower one is taken
        parent[3], parent[2] = 0, 0
        token[3] = token[2] = sampled[0] = 5
        token[1] = 4
    draft = rng.standard_normal((2, nl, nkv, n + 1, hd)).astype(elt)
    cache = rng.standard_normal((2, nl, nkv, max_seq, hd)).astype(elt)
    path, acc, step, got = run_commit(token, parent, sampled, past, draft, cache, kv)
    want = S.accepted(token, parent, sampled, max_seq - past if 0 <= past < max_seq else 0)
    assert acc == len(want) and list(path[:acc]) == want and (path[acc:] == -1).all()
    assert list(step) == ([sampled[want[-1]], past + acc] if want else [77, 77])
    for i, t in enumerate(want):
        cache[:, :, :, past + i] = draft[:, :, :, t]
    assert got.tobytes() == cache.tobytes()


def test_tree_commit_no_node():
    z = np.zeros((2, 1, 1, 4, 8), np.float32)
    path, acc, step, _ = run_commit([1, 1], [-2, 0], [1, 1], 0, z[:, :, :, :2], z, 0)
    assert acc == 0 and list(path) == [-1, -1] and list(step) == [77, 77]


# ----------------------------------------------------------------------------------- a step of them

class Step:
    """The four operators of one step over one layer, from inputs that the host writes: rotary positions, attention, tokens
    from given logits, the commit. Sizes that take every kernel's longer path."""
    N, NH, NKV, HD, VOCAB, MAX = 20, 8, 2, 64, 4133, 400

    def __init__(self, scratch=None):
        n, nh, nkv, hd, vocab, mx = self.N, self.NH, self.NKV, self.HD, self.VOCAB, self.MAX
        L = lib()
        self.width = (nh + 2 * nkv) * hd
        self.b = {k: up(np.zeros(v, t)) for k, (v, t) in dict(
            x=((n, self.width), np.float32), pos=(n, np.int32), node=(n, np.int32), parent=(n, np.int32), past=(1, np.int32),
            logits=((n, vocab), np.float32), temp=(n, np.float32), top_k=(n, np.int32), top_p=(n, np.float32),
            u=(n, np.float32), token=(n, np.int32), cache=((2, nkv, mx, hd), np.float16)).items()}
        self.o = {k: up(np.zeros(v, t)) for k, (v, t) in dict(
            q=((n, nh * hd), np.float32), draft=((2, nkv, n, hd), np.float16), out=((n, nh * hd), np.float32),
            sampled=(n, np.int32), prob=(n, np.float32), path=(n, np.int32), n_acc=(1, np.int32), step=(2, np.int32)).items()}
        self.like = {"q": np.float32, "draft": np.uint16, "out": np.float32, "sampled": np.int32, "prob": np.float32,
                     "path": np.int32, "n_acc": np.int32, "step": np.int32}
        floats, ws = L.sdy_attn_tree_floats(n, nh, nkv, hd, mx), L.sdy_sample_ws_bytes(n, vocab)
        self.scratch = scratch or (capi.DeviceBuffer(4 * floats), capi.DeviceBuffer(ws))
        self.freq = up(rope_freq(hd)[0])
        b, o = {k: v.ptr for k, v in self.b.items()}, {k: v.ptr for k, v in self.o.items()}
        half, dhalf = nkv * mx * hd * 2, nkv * n * hd * 2
        self.calls = [
            (L.sdy_qk_rope_at, capi.SdyRopeAtArgs(
                q=b["x"], k=b["x"] + 4 * nh * hd, v=b["x"] + 4 * (nh + nkv) * hd, q_stride=self.width, k_stride=self.width,
                v_stride=self.width, q_out=o["q"], q_out_stride=nh * hd, k_rows=o["draft"], v_rows=o["draft"] + dhalf,
                head_stride=n * hd, kv_type=1, n_slot=n, pos=b["pos"], slot=b["node"], freq=self.freq.ptr, mscale=1.0, n_rot=hd,
                n_tok=n, n_head=nh, n_kv_head=nkv, hd=hd)),
            (L.sdy_attn_tree, capi.SdyAttnTreeArgs(
                q=o["q"], q_stride=nh * hd, k_cache=b["cache"], v_cache=b["cache"] + half, head_stride=mx * hd,
                k_draft=o["draft"], v_draft=o["draft"] + dhalf, draft_stride=n * hd, kv_type=1, parent=b["parent"],
                n_past=b["past"], max_past=mx, n_tok=n, n_head=nh, n_kv_head=nkv, hd=hd, out=o["out"], out_stride=nh * hd,
                part=self.scratch[0].ptr)),
            (L.sdy_sample, capi.SdySampleArgs(
                logits=b["logits"], stride=vocab, n_rows=n, n_vocab=vocab, temp=b["temp"], top_k=b["top_k"], top_p=b["top_p"],
                u=b["u"], token=o["sampled"], prob=o["prob"], ws=self.scratch[1].ptr)),
            (L.sdy_tree_commit, capi.SdyTreeCommitArgs(
                token=b["token"], parent=b["parent"], sampled=o["sampled"], n_tok=n, n_past=b["past"], k_draft=o["draft"],
                v_draft=o["draft"] + dhalf, draft_stride=n * hd, draft_layer_stride=nkv * n * hd, k_cache=b["cache"],
                v_cache=b["cache"] + half, head_stride=mx * hd, layer_stride=nkv * mx * hd, kv_type=1, max_seq=mx, n_layer=1,
                n_kv_head=nkv, hd=hd, path=o["path"], n_acc=o["n_acc"], step=o["step"]))]

    def fill(self, seed, stream=None):
        rng = np.random.default_rng(seed)
        n = self.N
        parent = S.random_tree(n, rng, unused=int(rng.integers(0, 5)))
        past = int(rng.integers(0, self.MAX))
        logits = np.round(rng.standard_normal((n, self.VOCAB)) * 4).astype(np.float32)
        new = dict(x=rng.standard_normal((n, self.width)), pos=past + S.ancestors(parent).sum(1), node=np.arange(n),
                   parent=parent, past=[past], logits=logits, temp=rng.choice([0, 0.7, 2], n), top_k=rng.choice([0, 40], n),
                   top_p=rng.choice([1, 0.9], n), u=rng.random(n), token=np.argmax(logits, 1)[np.maximum(parent, 0)],
                   cache=rng.standard_normal((2, self.NKV, self.MAX, self.HD)))
        types = dict(x=np.float32, pos=np.int32, node=np.int32, parent=np.int32, past=np.int32, logits=np.float32,
                     temp=np.float32, top_k=np.int32, top_p=np.float32, u=np.float32, token=np.int32, cache=np.float16)
        self.sent = {k: np.ascontiguousarray(v, types[k]) for k, v in new.items()}
        for k, v in self.sent.items():
            assert v.nbytes == self.b[k].nbytes
            capi.check(lib().sdy_h2d(self.b[k].ptr, v.ctypes.data, v.nbytes, stream))
        for v in self.o.values():  # (an empty place's output row stays as it was)
            capi.check(lib().sdy_memset(v.ptr, 0, v.nbytes, stream))
        return self

    def run(self, stream=None):
        for fn, a in self.calls:
            capi.check(fn(ctypes.byref(a), stream))

    def got(self, stream=None):
        got = {k: v.to_array(self.like[k], v.nbytes // np.dtype(self.like[k]).itemsize, stream) for k, v in self.o.items()}
        got["cache"] = self.b["cache"].to_array(np.uint16, self.b["cache"].nbytes // 2, stream)
        return got


def same(a, b):
    return all(np.array_equal(a[k].view(np.uint16), b[k].view(np.uint16)) for k in a)


def test_a_recorded_step_replays_for_other_trees():
    """Two recorded steps on one scratch, replayed in turn with new inputs, eager steps between: the eager step's bits."""
    L = lib()
    st = ctypes.c_void_p()
    capi.check(L.sdy_stream_new(ctypes.byref(st)))
    eager = Step()
    steps = [Step()]
    steps.append(Step(steps[0].scratch))
    graphs = []
    for x in steps:
        x.fill(0).run()  # (what a first launch sets up is not recorded)
        capi.check(L.sdy_sync(None))
        capi.check(L.sdy_graph_begin(st))
        x.run(st)
        g = ctypes.c_void_p()
        capi.check(L.sdy_graph_end(st, ctypes.byref(g)))
        graphs.append(g)
    taken = set()
    for k in range(12):
        x, g = steps[k % 2], graphs[k % 2]
        x.fill(100 + k, st)
        capi.check(L.sdy_graph_launch(g, st))
        eager.fill(100 + k).run()
        want = eager.got()
        assert same(x.got(st), want), k
        taken.add(int(want["n_acc"][0]))
    assert len(taken) > 1
    for g in graphs:
        capi.check(L.sdy_graph_free(g))
    capi.check(L.sdy_stream_free(st))


def test_steps_on_two_streams_at_once():
    """Each with its own scratch."""
    L = lib()
    sts = [ctypes.c_void_p() for _ in range(2)]
    for st in sts:
        capi.check(L.sdy_stream_new(ctypes.byref(st)))
    steps, eager = [Step(), Step()], Step()
    for k in range(4):
        for i, (x, st) in enumerate(zip(steps, sts)):
            x.fill(10 * k + i, st)
        for x, st in zip(steps, sts):
            x.run(st)
        for i, (x, st) in enumerate(zip(steps, sts)):
            got = x.got(st)
            eager.fill(10 * k + i).run()
            assert same(got, eager.got()), (k, i)
    for st in sts:
        capi.check(L.sdy_stream_free(st))


def test_rows_beyond_32_bit_offsets():
    """Heads 2^31 elements apart: rotated rows written there, attended to, and moved there by the commit."""
    n, past, hd, far, rng = 6, 45, 128, (1 << 31) + 128, np.random.default_rng(8)
    big = [capi.DeviceBuffer(2 * (far + 64 * hd)) for _ in range(2)]  # f16
    t = Tree(n, past, 4, 2, hd, 1, 5)
    for buf, rows in zip(big, t.cache):
        for g in range(2):
            r = np.ascontiguousarray(rows[g, :past])
            capi.check(lib().sdy_h2d(buf.ptr + 2 * g * far, r.ctypes.data, r.nbytes, None))
    capi.check(lib().sdy_sync(None))
    t.args.k_cache, t.args.v_cache, t.args.head_stride, t.args.max_past = big[0].ptr, big[1].ptr, far, past
    t.part = capi.DeviceBuffer(4 * lib().sdy_attn_tree_floats(n, 4, 2, hd, past))
    t.args.part = t.part.ptr
    t.run().check()
    # the commit of the first two nodes behind them
    ints = [up(np.array(x, np.int32)) for x in ([3] * n, [-1, 0] + [-2] * (n - 2), [3] * n, [past], [0] * n, [0], [0, 0])]
    p = [b.ptr for b in ints]
    c = capi.SdyTreeCommitArgs(token=p[0], parent=p[1], sampled=p[2], n_tok=n, n_past=p[3], k_draft=t.args.k_draft,
                               v_draft=t.args.v_draft, draft_stride=n * hd, draft_layer_stride=2 * n * hd, k_cache=big[0].ptr,
                               v_cache=big[1].ptr, head_stride=far, layer_stride=2 * far, kv_type=1, max_seq=64, n_layer=1,
                               n_kv_head=2, hd=hd, path=p[4], n_acc=p[5], step=p[6])
    capi.check(lib().sdy_tree_commit(ctypes.byref(c), None))
    # and rotary rows to the next position
    x, freq = rng.standard_normal((1, 3 * 2 * hd)).astype(np.float32), rope_freq(hd)[0]
    bx, bf, bp, bq = up(x), up(freq), up(np.array([past + 2], np.int32)), capi.DeviceBuffer(4 * 2 * hd)
    a = capi.SdyRopeAtArgs(q=bx.ptr, k=bx.ptr + 8 * hd, v=bx.ptr + 16 * hd, q_stride=6 * hd, k_stride=6 * hd, v_stride=6 * hd,
                           q_out=bq.ptr, q_out_stride=2 * hd, k_rows=big[0].ptr, v_rows=big[1].ptr, head_stride=far, kv_type=1,
                           n_slot=64, pos=bp.ptr, freq=bf.ptr, mscale=1.0, n_rot=hd, n_tok=1, n_head=2, n_kv_head=2, hd=hd)
    capi.check(lib().sdy_qk_rope_at(ctypes.byref(a), None))
    for i, buf in enumerate(big):
        for g in range(2):
            got = np.empty((3, hd), np.float16)
            capi.check(lib().sdy_d2h(got.ctypes.data, buf.ptr + 2 * (g * far + past * hd), got.nbytes, None))
            capi.check(lib().sdy_sync(None))
            assert np.array_equal(got[:2].view(np.uint16), t.draft[i][g, :2].view(np.uint16))
            if i:
                assert np.array_equal(got[2], x[0, (4 + g) * hd:(5 + g) * hd].astype(np.float16))
            else:
                want, tol = S.rope(x[:, (2 + g) * hd:(3 + g) * hd][:, None], np.array([past + 2]), freq, 1.0, hd, 0)
                assert (np.abs(got[2] - want[0, 0]) <= tol[0, 0] + S.U16 * np.abs(want[0, 0]) * 1.01 + 2.0 ** -25).all()


@pytest.mark.parametrize("kv", [0, 1], ids=["f32", "f16"])
def test_attn_tree_very_long_cache(kv):
    """18 million positions: 2.3 or 4.6 GB of K. All K rows are 0 but the last one, whose weight is about that of all others."""
    past, hd, elt = 18_000_001, 64, (np.float32, np.float16)[kv]
    L = lib()
    nbytes = past * hd * np.dtype(elt).itemsize
    cache = [capi.DeviceBuffer(nbytes) for _ in range(2)]
    for c in cache:
        capi.check(L.sdy_memset(c.ptr, 0, nbytes, None))
    q = np.zeros((1, 1, hd), np.float32)
    q[0, 0, 0] = 8.0
    last = np.zeros((2, hd), elt)
    last[0, 0] = 16.75  # the score 8 * 16.75 / sqrt(64)
    last[1] = 1 + np.arange(hd)
    first = np.full(hd, 512, elt)
    at = nbytes - hd * last.itemsize
    for c, x in zip(cache, last):
        capi.check(L.sdy_h2d(c.ptr + at, x.ctypes.data, x.nbytes, None))
    capi.check(L.sdy_h2d(cache[1].ptr, first.ctypes.data, first.nbytes, None))
    capi.check(L.sdy_sync(None))
    b = [up(x) for x in (q, np.zeros((1, hd), elt), np.zeros((1, hd), elt), np.array([-1], np.int32), np.array([past], np.int32),
                         np.zeros(hd, np.float32))]
    part = capi.DeviceBuffer(4 * L.sdy_attn_tree_floats(1, 1, 1, hd, past))
    a = capi.SdyAttnTreeArgs(q=b[0].ptr, q_stride=hd, k_cache=cache[0].ptr, v_cache=cache[1].ptr, head_stride=past * hd,
                             k_draft=b[1].ptr, v_draft=b[2].ptr, draft_stride=hd, kv_type=kv, parent=b[3].ptr, n_past=b[4].ptr,
                             max_past=past, n_tok=1, n_head=1, n_kv_head=1, hd=hd, out=b[5].ptr, out_stride=hd, part=part.ptr)
    capi.check(L.sdy_attn_tree(ctypes.byref(a), None))
    w = np.exp(16.75)
    want = (w * last[1].astype(np.float64) + 512) / (past + w)  # (past - 1 zeros, the drafted row's and the last one)
    # the exponent's argument (24.2 in base 2, rounded twice, times ln 2) and exponential, the sums' parts (at most 600 of
    # them, a span's own sum of 16s is exact), the quotient
    tol = (2 * 24.2 * 0.7 + 2 + 600 + 2) * S.U32 * want
    assert (np.abs(b[5].to_array(np.float32, hd) - want) <= tol).all()


def test_a_step_answers_as_one_token_at_a_time():
    """Two attention layers' worth of a toy model, greedy: drafted trees checked by the four operators on the device give
    the tokens that one token at a time gives, whatever is drafted."""
    L = lib()
    rng = np.random.default_rng(12)
    nh, nkv, hd, vocab, n_layer, max_seq = 4, 2, 64, 97, 2, 64
    dim, width = nh * hd, (nh + 2 * nkv) * hd
    emb = rng.standard_normal((vocab, dim)).astype(np.float32)
    w = [(rng.standard_normal((dim, width)) / 16).astype(np.float32) for _ in range(n_layer)]
    head = rng.standard_normal((dim, vocab)).astype(np.float32)
    freq, mscale = rope_freq(hd)
    elt = 4
    cache = [capi.DeviceBuffer(n_layer * nkv * max_seq * hd * elt) for _ in range(2)]
    n_max = 9
    draft = [capi.DeviceBuffer(n_layer * nkv * n_max * hd * elt) for _ in range(2)]
    bfreq, bstep = up(freq), up(np.zeros(2, np.int32))
    layer = lambda b, l, rows: b.ptr + l * nkv * rows * hd * elt  # noqa: E731

    def forward(tokens, parent, past):
        """Logits of the nodes; their K/V rows are left in the draft's memory."""
        n = len(tokens)
        depth = S.ancestors(np.array(parent)).sum(1) - 1
        x = emb[tokens]
        bp, bpar, bpast = up((past + depth).astype(np.int32)), up(np.array(parent, np.int32)), up(np.array([past], np.int32))
        slots = up(np.arange(n, dtype=np.int32))
        for l in range(n_layer):
            bx, bq, bo = up(x @ w[l]), capi.DeviceBuffer(n * dim * 4), up(np.zeros((n, dim), np.float32))
            a = capi.SdyRopeAtArgs(q=bx.ptr, k=bx.ptr + 4 * dim, v=bx.ptr + 4 * (dim + nkv * hd), q_stride=width,
                                   k_stride=width, v_stride=width, q_out=bq.ptr, q_out_stride=dim,
                                   k_rows=layer(draft[0], l, n_max), v_rows=layer(draft[1], l, n_max),
                                   head_stride=n_max * hd, n_slot=n_max, pos=bp.ptr, slot=slots.ptr, freq=bfreq.ptr,
                                   mscale=mscale, n_rot=hd, n_tok=n, n_head=nh, n_kv_head=nkv, hd=hd)
            capi.check(L.sdy_qk_rope_at(ctypes.byref(a), None))
            part = capi.DeviceBuffer(4 * L.sdy_attn_tree_floats(n, nh, nkv, hd, max_seq))
            t = capi.SdyAttnTreeArgs(q=bq.ptr, q_stride=dim, k_cache=layer(cache[0], l, max_seq),
                                     v_cache=layer(cache[1], l, max_seq), head_stride=max_seq * hd, k_draft=a.k_rows,
                                     v_draft=a.v_rows, draft_stride=n_max * hd, parent=bpar.ptr, n_past=bpast.ptr,
                                     max_past=max_seq, n_tok=n, n_head=nh, n_kv_head=nkv, hd=hd, out=bo.ptr, out_stride=dim,
                                     part=part.ptr)
            capi.check(L.sdy_attn_tree(ctypes.byref(t), None))
            x = x + bo.to_array(np.float32, (n, dim))
        return x @ head

    def step(tokens, parent, past):
        n = len(tokens)
        logits = up(forward(tokens, parent, past))
        bt, ws = capi.DeviceBuffer(4 * n), capi.DeviceBuffer(L.sdy_sample_ws_bytes(n, vocab))
        bu, btemp = up(np.zeros(n, np.float32)), up(np.zeros(n, np.float32))
        capi.check(L.sdy_sample(ctypes.byref(capi.SdySampleArgs(
            logits=logits.ptr, stride=vocab, n_rows=n, n_vocab=vocab, temp=btemp.ptr, u=bu.ptr, token=bt.ptr, ws=ws.ptr)), None))
        ins = [up(np.array(z, np.int32)) for z in (tokens, parent, [past])]
        outs = [capi.DeviceBuffer(4 * n), capi.DeviceBuffer(4)]
        capi.check(L.sdy_tree_commit(ctypes.byref(capi.SdyTreeCommitArgs(
            token=ins[0].ptr, parent=ins[1].ptr, sampled=bt.ptr, n_tok=n, n_past=ins[2].ptr, k_draft=draft[0].ptr,
            v_draft=draft[1].ptr, draft_stride=n_max * hd, draft_layer_stride=nkv * n_max * hd, k_cache=cache[0].ptr,
            v_cache=cache[1].ptr, head_stride=max_seq * hd, layer_stride=nkv * max_seq * hd, max_seq=max_seq,
            n_layer=n_layer, n_kv_head=nkv, hd=hd, path=outs[0].ptr, n_acc=outs[1].ptr, step=bstep.ptr)), None))
        acc = int(outs[1].to_array(np.int32, 1)[0])
        path = outs[0].to_array(np.int32, n)[:acc]
        nxt, pos = bstep.to_array(np.int32, 2)
        assert pos == past + acc
        return [tokens[t] for t in path], int(nxt), int(pos)

    one, tok, past = [], 3, 0
    while past < 40:
        took, tok, past = step([tok], [-1], past)
        one += took
    tree, tok, past, steps = [], 3, 0, 0
    while past < 40:
        # right drafts (known from the first run) among wrong ones
        right = one[past + 1:past + 4] + [0] * 3
        tokens = [tok, (right[0] + 1) % vocab, right[0], right[1], (right[1] + 3) % vocab, right[2], 1, 2, 3]
        took, tok, past = step(tokens, [-1, 0, 0, 2, 2, 3, 5, -2, -2], past)
        tree += took
        steps += 1
    assert tree[:40] == one[:40] and steps <= 14
