"""The speculative-decoding entry points without a GPU: every refusal comes before anything is launched, and the
frequencies of scaled rotary positions (made on the host) against their published formulas."""
import ctypes
import math

import numpy as np
import pytest

from sardyne_amd import capi

P = 0x10000  # an address that a refused call never reads


def refused(fn, args, word):
    assert fn(ctypes.byref(args), None) == -1
    assert word in capi.lib().sdy_last_error().decode()


def rope_args(**kw):
    a = dict(q=P, k=P, v=P, q_stride=512, k_stride=128, v_stride=128, q_out=2 * P, q_out_stride=512, k_rows=P, v_rows=P,
             head_stride=64 * 9, kv_type=0, n_slot=9, pos=P, slot=P, freq=P, mscale=1.0, n_rot=64, interleaved=0, eps=1e-6,
             n_tok=3, n_head=8, n_kv_head=2, hd=64)
    return capi.SdyRopeAtArgs(**{**a, **kw})


@pytest.mark.parametrize("kw,word", [
    (dict(hd=63), "head_dim"), (dict(hd=514), "head_dim"), (dict(n_rot=66), "n_rot"), (dict(n_rot=31), "n_rot"),
    (dict(n_rot=-2), "n_rot"), (dict(kv_type=2), "KV type"), (dict(q=None, k=None), "neither"), (dict(pos=None), "pos"),
    (dict(freq=None), "freq"), (dict(q_out=None), "q_out"), (dict(n_head=0), "n_head"), (dict(v=None), "v,"),
    (dict(k_rows=None), "k_rows"), (dict(v_rows=None), "v_rows"), (dict(n_kv_head=0), "n_kv_head"),
    (dict(head_stride=64 * 9 - 1), "stride"), (dict(n_slot=-1), "slots"), (dict(n_tok=-1), "n_tok"),
    (dict(q_out=P, q_out_stride=516), "in place"), (dict(q_out_stride=511), "apart")])
def test_rope_at_refusals(kw, word):
    refused(capi.lib().sdy_qk_rope_at, rope_args(**kw), word)


def tree_args(**kw):
    a = dict(q=P, q_stride=512, k_cache=P, v_cache=P, head_stride=64 * 50, k_draft=P, v_draft=P, draft_stride=64 * 5,
             kv_type=0, parent=P, n_past=P, max_past=50, n_tok=5, n_head=8, n_kv_head=2, hd=64, out=P, out_stride=512,
             part=P)
    return capi.SdyAttnTreeArgs(**{**a, **kw})


@pytest.mark.parametrize("kw,word", [
    (dict(n_tok=257), "n_tok"), (dict(n_tok=-1), "n_tok"), (dict(n_head=7), "multiple"), (dict(n_kv_head=0), "multiple"),
    (dict(hd=96), "head_dim"), (dict(kv_type=3), "KV type"), (dict(q=None), "needed"), (dict(k_draft=None), "needed"),
    (dict(v_draft=None), "needed"), (dict(parent=None), "needed"), (dict(n_past=None), "needed"), (dict(out=None), "needed"),
    (dict(part=None), "needed"), (dict(max_past=-1), "max_past"), (dict(max_past=(1 << 28) + 1, head_stride=1 << 40), "max_past"), (dict(k_cache=None), "cache"), (dict(v_cache=None), "cache"),
    (dict(head_stride=64 * 49), "next one"), (dict(draft_stride=64 * 4), "next one"), (dict(q=P + 4), "aligned"),
    (dict(out=P + 8), "aligned"), (dict(q_stride=514), "aligned"), (dict(out_stride=513), "aligned"),
    (dict(k_cache=P + 2), "aligned"), (dict(kv_type=1, head_stride=64 * 50 + 4), "aligned"), (dict(q_stride=508), "rows of"),
    (dict(out_stride=508), "rows of")])
def test_attn_tree_refusals(kw, word):
    refused(capi.lib().sdy_attn_tree, tree_args(**kw), word)


def test_attn_tree_sizes():
    lib = capi.lib()
    assert lib.sdy_attn_tree_ok(256, 64, 1, 256) == 1 and lib.sdy_attn_tree_ok(1, 1, 1, 64) == 1
    assert lib.sdy_attn_tree_ok(0, 8, 2, 64) == lib.sdy_attn_tree_ok(5, 8, 3, 64) == lib.sdy_attn_tree_ok(5, 8, 2, 80) == 0
    assert lib.sdy_attn_tree_floats(0, 8, 2, 64, 100) == lib.sdy_attn_tree_floats(5, 8, 2, 64, -1) == 0
    assert lib.sdy_attn_tree_floats(5, 8, 2, 64, 0) > 0
    small, large = lib.sdy_attn_tree_floats(64, 32, 4, 128, 1000), lib.sdy_attn_tree_floats(64, 32, 4, 128, 100000)
    assert 0 < small <= large


def sample_args(**kw):
    a = dict(logits=P, stride=100, n_rows=3, n_vocab=100, u=P, token=P, ws=P)
    return capi.SdySampleArgs(**{**a, **kw})


@pytest.mark.parametrize("kw,word", [
    (dict(n_rows=-1), "n_rows"), (dict(n_rows=65536), "n_rows"), (dict(n_vocab=0), "n_vocab"), (dict(n_vocab=(1 << 22) + 1), "n_vocab"),
    (dict(stride=99), "apart"), (dict(logits=None), "needed"), (dict(u=None), "needed"), (dict(token=None), "needed"),
    (dict(ws=None), "needed"), (dict(ws=P + 8), "aligned")])
def test_sample_refusals(kw, word):
    refused(capi.lib().sdy_sample, sample_args(**kw), word)


def test_sample_ws_sizes():
    lib = capi.lib()
    assert lib.sdy_sample_ws_bytes(0, 10) == lib.sdy_sample_ws_bytes(1, 0) == lib.sdy_sample_ws_bytes(1, (1 << 22) + 1) == 0
    assert lib.sdy_sample_ws_bytes(1, 1) > 0


def commit_args(**kw):
    a = dict(token=P, parent=2 * P, sampled=3 * P, n_tok=4, n_past=4 * P, k_draft=P, v_draft=2 * P, draft_stride=256,
             draft_layer_stride=512, k_cache=3 * P, v_cache=4 * P, head_stride=640, layer_stride=1280, kv_type=0, max_seq=10,
             n_layer=2, n_kv_head=2, hd=64, path=5 * P, n_acc=6 * P, step=7 * P)
    return capi.SdyTreeCommitArgs(**{**a, **kw})


@pytest.mark.parametrize("kw,word", [
    (dict(n_tok=0), "n_tok"), (dict(n_tok=257), "n_tok"), (dict(kv_type=7), "KV type"), (dict(n_layer=0), "n_layer"),
    (dict(n_layer=65536), "n_layer"), (dict(hd=0), "head_dim"), (dict(hd=513), "head_dim"), (dict(max_seq=0), "max_seq"),
    (dict(n_kv_head=0), "n_kv_head")] + [
    ({k: None}, "needed") for k in ("token", "parent", "sampled", "n_past", "k_draft", "v_draft", "k_cache", "v_cache",
                                    "path", "n_acc", "step")] + [
    (dict(step=4 * P - 4), "overlap"), (dict(path=P), "overlap"), (dict(n_acc=2 * P + 12), "overlap"),
    (dict(path=3 * P - 12), "overlap"), (dict(k_draft=3 * P), "own"), (dict(v_draft=4 * P), "own"),
    (dict(k_draft=3 * P + 10 * 256 - 16), "own"), (dict(v_draft=4 * P - 4 * 256 + 16), "own"),
    (dict(n_acc=5 * P + 12), "overlap"), (dict(step=6 * P - 4), "overlap"), (dict(step=5 * P - 4), "overlap"),
    (dict(head_stride=639), "reach"), (dict(draft_stride=255), "reach"), (dict(layer_stride=1279), "reach"),
    (dict(draft_layer_stride=511), "reach")])
def test_tree_commit_refusals(kw, word):
    refused(capi.lib().sdy_tree_commit, commit_args(**kw), word)


def test_no_arguments():
    lib = capi.lib()
    for fn in (lib.sdy_qk_rope_at, lib.sdy_attn_tree, lib.sdy_sample, lib.sdy_tree_commit):
        assert fn(None, None) == -1


def test_speculate_without_a_context():
    one = (ctypes.c_int32 * 1)()
    n = ctypes.c_int32()
    assert capi.lib().sdy_engine_speculate(None, one, one, 1, None, None, one, ctypes.byref(n), ctypes.byref(n)) == -1


def test_empty_calls_do_nothing():
    lib = capi.lib()
    assert lib.sdy_qk_rope_at(ctypes.byref(rope_args(n_tok=0)), None) == 0
    assert lib.sdy_attn_tree(ctypes.byref(tree_args(n_tok=0)), None) == 0
    assert lib.sdy_sample(ctypes.byref(sample_args(n_rows=0)), None) == 0


# ------------------------------------------------------------------------------- frequencies

def freqs(n_rot, theta, **kw):
    f, m = np.full(max(n_rot // 2, 1), np.nan), ctypes.c_float()
    sc = capi.SdyRopeScaling(**kw) if kw else None
    rc = capi.lib().sdy_rope_freqs(f.ctypes.data, ctypes.byref(m), n_rot, theta, ctypes.byref(sc) if sc else None)
    return rc, f[:n_rot // 2], m.value


@pytest.mark.parametrize("n_rot,theta", [(0, 1e4), (2, 1e4), (64, 1e4), (128, 1e6), (122, 5e5)])
def test_rope_freqs_plain_and_linear(n_rot, theta):
    exp = np.array([1.0 / theta ** (2 * i / n_rot) for i in range(n_rot // 2)])
    rc, f, m = freqs(n_rot, theta)
    assert rc == 0 and m == 1.0 and np.allclose(f, exp, rtol=1e-14, atol=0)
    rc, f, m = freqs(n_rot, theta, kind=capi.ROPE_LINEAR, factor=4.0)
    assert rc == 0 and m == 1.0 and np.allclose(f, exp / 4, rtol=1e-14, atol=0)


@pytest.mark.parametrize("n_rot,theta,factor,orig", [(128, 1e6, 4.0, 32768), (64, 1e4, 16.0, 4096), (32, 1e4, 2.0, 128)])
def test_rope_freqs_yarn(n_rot, theta, factor, orig):
    rc, f, m = freqs(n_rot, theta, kind=capi.ROPE_YARN, factor=factor, orig_ctx=orig, beta_fast=32.0, beta_slow=1.0)
    assert rc == 0 and abs(m - (0.1 * math.log(factor) + 1)) < 1e-7

    def index(turns):  # of the pair that turns so many times over the original context
        return n_rot * math.log(orig / (turns * 2 * math.pi)) / (2 * math.log(theta))

    low, high = max(math.floor(index(32)), 0), min(math.ceil(index(1)), n_rot - 1)
    for i in range(n_rot // 2):
        base = theta ** (-2 * i / n_rot)
        r = min(max((i - low) / max(high - low, 1e-3), 0), 1)
        assert f[i] == pytest.approx(base / factor * r + base * (1 - r), rel=1e-13)
    rc, _, m = freqs(n_rot, theta, kind=capi.ROPE_YARN, factor=factor, orig_ctx=orig, beta_fast=32.0, beta_slow=1.0,
                     attn_factor=1.25)
    assert rc == 0 and m == 1.25


def test_rope_freqs_llama3():
    rc, f, m = freqs(128, 5e5, kind=capi.ROPE_LLAMA3, factor=8.0, orig_ctx=8192, low_freq=1.0, high_freq=4.0)
    assert rc == 0 and m == 1.0
    for i in range(64):
        base = 5e5 ** (-2 * i / 128)
        wave = 2 * math.pi / base
        if wave < 8192 / 4:
            exp = base
        elif wave > 8192:
            exp = base / 8
        else:
            smooth = (8192 / wave - 1) / 3
            exp = (1 - smooth) * base / 8 + smooth * base
        assert f[i] == pytest.approx(exp, rel=1e-13)


@pytest.mark.parametrize("n_rot,theta,kw", [
    (63, 1e4, {}), (-2, 1e4, {}), (514, 1e4, {}), (64, 1.0, {}), (64, math.inf, {}), (64, math.nan, {}),
    (64, 1e4, dict(kind=4, factor=2.0)), (64, 1e4, dict(kind=-1, factor=2.0)), (64, 1e4, dict(kind=1, factor=0.0)),
    (64, 1e4, dict(kind=1, factor=math.nan)), (64, 1e4, dict(kind=2, factor=2.0, beta_fast=32.0, beta_slow=1.0)),
    (64, 1e4, dict(kind=2, factor=2.0, orig_ctx=100, beta_fast=1.0, beta_slow=2.0)),
    (64, 1e4, dict(kind=3, factor=2.0, orig_ctx=100, low_freq=4.0, high_freq=4.0))])
def test_rope_freqs_refusals(n_rot, theta, kw):
    assert freqs(n_rot, theta, **kw)[0] == -1
