"""What the entry points for several candidates and bounded caches refuse
before they touch the GPU (these checks run without one)."""
import ctypes

import pytest

from gncx_b200 import core

INVALID, UNALIGNED = 1, 2
FAKE = 1 << 20  # never dereferenced: every call here is refused by its sizes


@pytest.fixture()
def lib():
    lib = core.load()
    lib.gncx_clear_error()
    yield lib
    lib.gncx_clear_error()


def tree(lib, pos0=4, n_tok=3, nh=4, nkv=2, hd=64):
    return lib.gncx_attention_tree(FAKE, FAKE, FAKE, FAKE, pos0, n_tok, nh, nkv, hd, 1.0, 0, FAKE, None, 0)


@pytest.mark.parametrize("bad", [dict(pos0=-1), dict(n_tok=0), dict(n_tok=-3), dict(n_tok=1025), dict(nh=3), dict(nkv=0),
                                 dict(nh=0), dict(hd=0), dict(hd=66), dict(hd=260), dict(pos0=2**31 - 2, n_tok=8),
                                 dict(pos0=2**30 - 7, n_tok=8), dict(nh=1025, nkv=1, n_tok=1024), dict(nkv=65536, nh=65536)])
def test_tree_refuses(lib, bad):
    assert tree(lib, **bad) == INVALID
    assert lib.gncx_last_error() == INVALID
    assert b"gncx_attention_tree" in lib.gncx_last_error_message()
    a = dict(pos0=4, n_tok=3, nh=4, nkv=2, hd=64) | bad
    assert lib.gncx_attention_tree_workspace(a["pos0"], a["n_tok"], a["nh"], a["nkv"], a["hd"], 0) == 0


@pytest.mark.parametrize("bad", [dict(pos=-1), dict(nh=3), dict(nkv=0), dict(hd=62), dict(hd=512), dict(stride=7),
                                 dict(pos=2**30, stride=2**31 - 1), dict(nh=65537, nkv=1)])
def test_step_refuses(lib, bad):
    a = dict(pos=7, nh=4, nkv=2, hd=64, stride=8) | bad
    assert lib.gncx_mqa_attention_step_weights(FAKE, FAKE, FAKE, FAKE, FAKE, a["pos"], a["pos"], a["nh"], a["nkv"], a["hd"],
                                               1.0, 1, FAKE, FAKE, FAKE, a["stride"], None, 0) == INVALID
    assert lib.gncx_last_error() == INVALID


@pytest.mark.parametrize("bad", [dict(rows=-1, keep=-1), dict(rows=2**30 + 1, stride=2**31 - 1), dict(keep=9), dict(keep=-1), dict(nkv=0), dict(hd=0), dict(hd=6),
                                 dict(stride=7), dict(out_stride=3), dict(pos=None), dict(pos_out=None),
                                 dict(w_out=FAKE), dict(pos_out=FAKE + 4096)])
def test_evict_refuses(lib, bad):
    a = dict(rows=8, keep=4, nkv=2, hd=64, stride=8, out_stride=4, pos=FAKE + 4096, pos_out=FAKE + 8192, w_out=FAKE + 64) | bad
    assert lib.gncx_kv_evict(FAKE, FAKE, FAKE, a["pos"], a["stride"], a["rows"], a["keep"], 0, a["nkv"], a["hd"], a["w_out"],
                             a["pos_out"], a["out_stride"], None, 0) == INVALID
    assert lib.gncx_last_error() == INVALID


def test_evict_workspace_grows_with_the_rows(lib):
    sizes = [lib.gncx_kv_evict_workspace(n, 64, 8) for n in (64, 65, 100, 1000, 100000)]
    assert sizes == sorted(sizes) and sizes[0] > 0
    assert lib.gncx_kv_evict_workspace(10, 11, 8) == 0


@pytest.mark.parametrize("bad", [dict(beams=0), dict(beams=257), dict(vocab=0), dict(vocab=(1 << 24) + 1), dict(n=0),
                                 dict(n=257), dict(eos=-1), dict(eos=1000)])
def test_beam_refuses(lib, bad):
    a = dict(beams=4, vocab=1000, n=8, eos=2) | bad
    assert lib.gncx_beam_select(FAKE, FAKE, FAKE, a["beams"], a["vocab"], a["eos"], a["n"], FAKE, FAKE, FAKE, FAKE, None,
                                0) == INVALID
    assert lib.gncx_last_error() == INVALID


@pytest.mark.parametrize("bad,code", [(dict(states=-1), INVALID), (dict(slots=-1), INVALID), (dict(slots=257), INVALID),
                                      (dict(n=62), UNALIGNED), (dict(slot=66), UNALIGNED), (dict(stride=258), UNALIGNED),
                                      (dict(n=1 << 40, slot=1 << 41), INVALID), (dict(stride=1 << 60), INVALID)])
def test_reorder_refuses(lib, bad, code):
    a = dict(states=2, stride=256, slots=4, slot=64, n=64) | bad
    assert lib.gncx_state_reorder(FAKE, a["states"], a["stride"], a["slots"], a["slot"], a["n"], FAKE) == code
    assert lib.gncx_last_error() == code


def test_needs_a_gpu(lib):
    torch = pytest.importorskip("torch")
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    assert tree(lib) == 4  # GNCX_ERR_NO_DEVICE
    assert lib.gncx_state_reorder(FAKE, 2, 256, 4, 64, 64, FAKE) == 4
    with pytest.raises(core.GncxError):
        core.check(lib)
