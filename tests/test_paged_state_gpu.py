"""States with a paged KV cache (vtb_cuda_state_create_paged): the forward loop
over pages against the contiguous cache and the oracle, forks that share pages,
windows that give pages back, compaction, and running out of pages."""
import numpy as np
import pytest

import oracle as O
from vantablack_b200 import _lib, ops, synth as S
from vantablack_b200.model import Context, CudaModel, CudaState, HostWeights, LlamaConfig, PagedConfig

pytestmark = pytest.mark.gpu

SMALL = LlamaConfig(dim=256, n_layers=2, n_heads=4, n_kv_heads=2, head_dim=64, ffn_dim=512, vocab_size=512, max_seq=128,
                    rope_base=10000.0)
LOGITS = 1e-3  # the bar of the forward loop against the oracle
# A 16-bit cache rounds q, k, v, p and the attention's output by half a step each, and a score by two more of
# its terms; over the two layers that stays below 16 half steps of the largest logit.
HALF_STEPS = {S.F16: 16 * 2.0 ** -11, S.BF16: 16 * 2.0 ** -8}


@pytest.fixture(scope="module")
def model():
    ctx = Context(0)
    w = HostWeights(SMALL, seed=5)
    m = CudaModel(ctx, w)
    yield m, w
    m.close()


def near(a, b, tol):
    return np.abs(a - b).max() <= tol * np.abs(b).max()


def tokens(n, seed=0):
    return np.random.default_rng(seed).integers(3, SMALL.vocab_size, n)


@pytest.mark.parametrize("page", [1, 16, 64, 256])
def test_paged_equals_contiguous(model, page):
    """Prompt in chunks, then decode through the graph and slot by slot."""
    m, _ = model
    plain, paged = CudaState(m, 1, 16), CudaState(m, 1, 16, paged=PagedConfig(-(-SMALL.max_seq // page), page))
    t = tokens(60, page)
    a, x = plain.prefill(t[:43])
    b, y = paged.prefill(t[:43])
    assert near(b, a, LOGITS) and x == y
    for i, tok in enumerate(t[43:]):
        (la, aa), (lb, ab) = plain.step([tok], graph=i % 3 != 0), paged.step([tok], graph=i % 3 != 0)
        assert near(lb, la, LOGITS) and np.array_equal(aa, ab)
    assert plain.pos() == paged.pos() == 60
    ops.check_device_error()


def test_paged_against_the_oracle(model):
    m, w = model
    ref, paged = O.Model(w), CudaState(m, 1, 32, paged=PagedConfig(6, 16))
    t = tokens(45, 2)
    a, (b, y) = ref.prefill(t[:33]), paged.prefill(t[:33])
    assert near(b, a, LOGITS) and y == O.argmax(a)
    for tok in t[33:]:
        a, (b, y) = ref.step(int(tok)), paged.step([int(tok)])
        assert near(b[0], a, LOGITS) and y[0] == O.argmax(a)
    ops.check_device_error()


@pytest.mark.parametrize("kv_type", [S.F16, S.BF16])
def test_sixteen_bit_caches(model, kv_type):
    m, _ = model
    plain, paged = CudaState(m, 2, 64), CudaState(m, 2, 64, paged=PagedConfig(40, 16, kv_type))
    t = tokens(50, 3)
    for s, n in ((0, 40), (1, 7)):
        a, b = plain.prefill(t[:n], s)[0], paged.prefill(t[:n], s)[0]
        assert near(b, a, HALF_STEPS[kv_type])
    for i in range(9):
        tok = [int(t[40 + i]), int(t[7 + i])]
        assert near(paged.step(tok)[0], plain.step(tok)[0], HALF_STEPS[kv_type])
    ops.check_device_error()


def test_fork_release_compact(model):
    """Three continuations of one prompt share its pages; a compaction in between changes nothing."""
    m, _ = model
    plain, paged = CudaState(m, 3, 64), CudaState(m, 3, 64, paged=PagedConfig(14, 16))
    t = tokens(39, 8)
    for s in range(3):
        plain.prefill(t, s)
    assert paged.free_pages() == 14
    paged.prefill(t, 0)
    assert paged.free_pages() == 11                  # 39 positions: two whole pages and 7 slots
    paged.fork(1, 0)
    paged.fork(2, 0)
    assert paged.free_pages() == 9                   # a private tail page each
    assert [paged.pos(s) for s in range(3)] == [39] * 3
    rng = np.random.default_rng(1)
    for i in range(25):
        tok = rng.integers(3, SMALL.vocab_size, 3)
        la, aa = plain.step(tok)
        lb, ab = paged.step(tok)
        for s in range(3):
            assert near(lb[s], la[s], LOGITS) and aa[s] == ab[s]
        if i == 12:
            paged.fork(1, 2)                         # over a sequence that holds pages
            plain.reset()
            break
    # after the second fork sequence 1 is a copy of 2
    tok = rng.integers(3, SMALL.vocab_size, 3)
    tok[1] = tok[2]
    l, a = paged.step(tok)
    assert near(l[1], l[2], 1e-4) and a[1] == a[2]
    free = paged.free_pages()
    paged.release(0)
    assert paged.pos(0) == 0 and paged.free_pages() > free
    live = paged.compact()
    assert live == 14 - paged.free_pages()
    tok = rng.integers(3, SMALL.vocab_size, 3)
    tok[1] = tok[2]
    l, a = paged.step(tok)
    assert near(l[1], l[2], 1e-4) and a[1] == a[2]
    paged.reset()
    assert paged.free_pages() == 14 and paged.compact() == 0
    ops.check_device_error()


def test_compaction_keeps_the_sequences(model):
    m, _ = model
    plain, paged = CudaState(m, 2, 64), CudaState(m, 2, 64, paged=PagedConfig(16, 8))
    t = tokens(60, 9)
    for st in (plain, paged):
        st.prefill(t[:50], 0)
        st.prefill(t[:21], 1)
    paged.release(0)                                  # holes before sequence 1's pages
    assert paged.compact() == 3
    plain.reset()
    plain.prefill(t[:21], 1)
    for i in range(6):
        tok = [int(t[i]), int(t[30 + i])]
        la, lb = plain.step(tok)[0], paged.step(tok)[0]
        assert near(lb[0], la[0], LOGITS) and near(lb[1], la[1], LOGITS)
    ops.check_device_error()


@pytest.mark.parametrize("window,sinks", [(24, 0), (24, 4), (40, 17), (1000, 3)])
def test_window(model, window, sinks):
    """Decode token by token, with pages given back on the way, equals a windowed prefill of the same tokens, and a
    window longer than the sequence equals none."""
    m, _ = model
    t = tokens(100, window)
    pc = PagedConfig(20, 8, S.F32, window, sinks)
    one, all_ = CudaState(m, 1, 128, paged=pc), CudaState(m, 1, 128, paged=pc)
    one.prefill(t[:5])
    for i in range(5, 100):
        la, _ = one.step([int(t[i])])
        kept = sum(1 for p in range(0, i + 1, 8) if p < sinks or p + 8 > i + 2 - window)
        assert 20 - one.free_pages() == kept
        if i in (30, 63, 99):
            all_.reset()
            lb, _ = all_.prefill(t[:i + 1])
            assert near(la[0], lb, LOGITS)
    if window >= 100:
        plain = CudaState(m, 1, 128)
        assert near(lb, plain.prefill(t)[0], LOGITS)
    ops.check_device_error()


def test_out_of_pages(model):
    """A step or prefill without pages fails with -7, changes nothing, and goes through once pages are free."""
    m, _ = model
    st, ref = CudaState(m, 2, 64, paged=PagedConfig(4, 16)), CudaState(m, 2, 64)
    t = tokens(70, 4)
    for s in (st, ref):
        s.prefill(t[:32], 0)
        s.prefill(t[:17], 1)
    assert st.free_pages() == 0
    with pytest.raises(_lib.VtbError) as e:
        st.step([5, 6])
    assert e.value.status == -7 and st.pos(0) == 32 and st.pos(1) == 17 and st.free_pages() == 0
    with pytest.raises(_lib.VtbError):
        st.prefill(t[:1], 0)
    st.release(0)
    st.prefill(t[:3], 0)
    ref.reset()
    ref.prefill(t[:3], 0)
    ref.prefill(t[:17], 1)
    la, lb = ref.step([9, 10])[0], st.step([9, 10])[0]
    assert near(lb, la, LOGITS)
    ops.check_device_error()


def test_fork_without_a_free_page(model):
    m, _ = model
    st = CudaState(m, 3, 64, paged=PagedConfig(3, 16))
    st.prefill(tokens(20, 1), 0)
    st.prefill(tokens(9, 2), 1)
    with pytest.raises(_lib.VtbError) as e:
        st.fork(2, 0)
    assert e.value.status == -7 and st.pos(2) == 0
    st.fork(1, 0)                                     # its own page serves the copy
    assert st.pos(1) == 20 and st.free_pages() == 0


def test_bad_paged_calls(model):
    m, _ = model
    for bad in (PagedConfig(0), PagedConfig(4, 12), PagedConfig(4, 2048), PagedConfig(4, 16, S.Q8_0), PagedConfig(4, 16, S.F32, -1),
                PagedConfig(4, 16, S.F32, 0, 2)):
        with pytest.raises(_lib.VtbError):
            CudaState(m, 1, 16, paged=bad)
    st, plain = CudaState(m, 2, 16, paged=PagedConfig(8, 16)), CudaState(m, 2, 16)
    assert plain.free_pages() == -1
    for call in (lambda: st.fork(0, 0), lambda: st.fork(2, 0), lambda: st.fork(0, -1), lambda: st.release(2), lambda: plain.fork(0, 1),
                 lambda: plain.release(0), lambda: plain.compact()):
        with pytest.raises(_lib.VtbError):
            call()
    st.lib.vtb_cuda_begin_token(st.h, np.array([4, 5], np.int32).ctypes.data)
    with pytest.raises(_lib.VtbError):  # a token is being computed
        st.release(0)
    st.reset()
    assert st.free_pages() == 8


def test_fork_shares_only_written_pages(model):
    """A begun token that is given up leaves its page with the sequence; a fork must not share it."""
    m, _ = model
    st, want = CudaState(m, 2, 64, paged=PagedConfig(16, 16)), CudaState(m, 2, 64, paged=PagedConfig(16, 16))
    for s in (st, want):
        s.prefill(tokens(16, 1), 1)                   # whole pages: the next token opens one
    st.lib.vtb_cuda_begin_token(st.h, np.array([4, 5], np.int32).ctypes.data)
    st.prefill(tokens(3, 2), 0)                       # ends the begun token
    for s in (st, want):
        s.fork(0, 1)
    for i in range(4):
        t = np.array([7 + i, 90 + i], np.int32)       # the two go on differently
        la, _ = st.step(t)
        lb, _ = want.step(t)
        assert np.array_equal(la, lb)
    assert not np.array_equal(la[0], la[1])
    ops.check_device_error()


def test_bad_token_in_a_later_chunk(model):
    """The chunks before it count, and the state goes on from there."""
    m, _ = model
    st, want = CudaState(m, 2, 16, paged=PagedConfig(16, 16)), CudaState(m, 2, 16, paged=PagedConfig(16, 16))
    t = tokens(40, 3)
    want.prefill(t[:16], 0)
    t[20] = SMALL.vocab_size
    with pytest.raises(_lib.VtbError):
        st.prefill(t, 0)
    assert st.pos(0) == 16
    st.fork(1, 0)                                     # nothing is being computed
    want.fork(1, 0)
    la, lb = st.step(np.array([5, 6], np.int32))[0], want.step(np.array([5, 6], np.int32))[0]
    assert np.array_equal(la, lb)
    st.release(0)
    assert st.pos(0) == 0
