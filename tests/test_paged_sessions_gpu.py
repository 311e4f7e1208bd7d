"""Sessions on a paged state: a windowed prompt behind queued work, prompts in chunks under a window, sequences that
stay idle, and calls that are refused in the middle of a token."""
import numpy as np
import pytest

import oracle as O
from vantablack_b200 import _lib, ops, synth as S
from vantablack_b200.model import Context, CudaModel, CudaState, HostWeights, LlamaConfig, PagedConfig

pytestmark = pytest.mark.gpu

SMALL = LlamaConfig(dim=256, n_layers=2, n_heads=4, n_kv_heads=2, head_dim=64, ffn_dim=512, vocab_size=512, max_seq=128,
                    rope_base=10000.0)
WIDE = LlamaConfig(dim=512, n_layers=2, n_heads=4, n_kv_heads=2, head_dim=128, ffn_dim=512, vocab_size=512, max_seq=128,
                   rope_base=10000.0)
TALL = LlamaConfig(dim=256, n_layers=2, n_heads=4, n_kv_heads=2, head_dim=64, ffn_dim=512, vocab_size=32768, max_seq=128,
                   rope_base=10000.0)
LOGITS = 1e-3  # the bar of the forward loop against the oracle


def make(cfg):
    m = CudaModel(Context(0), HostWeights(cfg, seed=5))
    yield m
    m.close()


@pytest.fixture(scope="module")
def model():
    yield from make(SMALL)


def near(a, b, tol):
    return np.abs(a - b).max() <= tol * np.abs(b).max()


def tokens(n, seed=0):
    return np.random.default_rng(seed).integers(3, SMALL.vocab_size, n)


def begin(st, toks):
    return st.lib.vtb_cuda_begin_token(st.h, np.array(toks, np.int32).ctypes.data)


@pytest.fixture(scope="module")
def tall():
    yield from make(TALL)


def test_windowed_prompt_behind_queued_work(tall):
    """The page table goes to the device while milliseconds of work are queued before it; pages that the window leaves
    at the end of the call are given back only when the table has been read."""
    n = 512
    pc = PagedConfig(n + 32, 8, S.F32, 24, 4)
    st, want = CudaState(tall, n, n, paged=pc), CudaState(tall, 1, 128, paged=pc)
    t = np.random.default_rng(3).integers(3, TALL.vocab_size, 100)
    a, x = want.prefill(t)
    assert begin(st, [5] * n) == 0
    for _ in range(200):  # given up: about 30 us each on the device, queued faster than that
        assert st.lib.vtb_cuda_final_step(st.h) == 0
    b, y = st.prefill(t)
    ops.check_device_error()
    assert near(b, a, LOGITS) and x == y


@pytest.mark.parametrize("kv_type", [S.F32, S.BF16])
@pytest.mark.parametrize("page,window,sinks", [(8, 24, 0), (8, 24, 9), (16, 50, 4), (1, 17, 1)])
def test_windowed_prompt_in_chunks(model, kv_type, page, window, sinks):
    """A prompt in chunks of 16 rows, with pages given back between them, equals one chunk, and the steps after it."""
    t = tokens(110, page + window)
    pc = PagedConfig(-(-128 // page), page, kv_type, window, sinks)
    one, cut = CudaState(model, 1, 128, paged=pc), CudaState(model, 1, 16, paged=pc)
    tol = LOGITS if kv_type == S.F32 else 16 * 2.0 ** -8
    a, b = one.prefill(t[:100])[0], cut.prefill(t[:100])[0]
    assert near(b, a, tol) and cut.free_pages() == one.free_pages()
    for tok in t[100:]:
        assert near(cut.step([tok])[0], one.step([tok])[0], tol)
    ops.check_device_error()


def test_head_dim_128_against_the_oracle():
    w = HostWeights(WIDE, seed=6)
    m = CudaModel(Context(0), w)
    ref, st = O.Model(w), CudaState(m, 1, 32, paged=PagedConfig(6, 16))
    t = tokens(45, 2)
    a, (b, y) = ref.prefill(t[:33]), st.prefill(t[:33])
    assert near(b, a, LOGITS) and y == O.argmax(a)
    for tok in t[33:]:
        a, (b, y) = ref.step(int(tok)), st.step([int(tok)])
        assert near(b[0], a, LOGITS) and y[0] == O.argmax(a)
    ops.check_device_error()
    m.close()


@pytest.mark.parametrize("graph", [True, False])
@pytest.mark.parametrize("kv_type", [S.F32, S.BF16])
def test_idle_sequences(model, kv_type, graph):
    """Token -1 leaves a sequence out of a step: it takes no page, keeps its position, and the others are as alone."""
    tol = LOGITS if kv_type == S.F32 else 16 * 2.0 ** -8
    st = CudaState(model, 3, 64, paged=PagedConfig(20, 8, kv_type))
    alone = [CudaState(model, 1, 64, paged=PagedConfig(20, 8, kv_type)) for _ in range(3)]
    t = tokens(200, 12)
    for s, n in ((0, 20), (1, 31), (2, 5)):
        st.prefill(t[:n], s)
        alone[s].prefill(t[:n])
    at = 40

    def step(active):
        nonlocal at
        toks = [int(t[at + s]) if s in active else -1 for s in range(3)]
        at += 3
        before = [st.pos(s) for s in range(3)]
        logits, arg = st.step(toks, graph=graph)
        for s in range(3):
            if s in active:
                la, aa = alone[s].step([toks[s]])
                assert near(logits[s], la[0], tol) and (kv_type != S.F32 or arg[s] == aa[0])
                assert st.pos(s) == before[s] + 1
            else:
                assert st.pos(s) == before[s] and arg[s] == -1

    step({0, 1, 2})
    st.release(1)
    held = 20 - st.free_pages() - sum(-(-st.pos(s) // 8) for s in (0, 2))
    assert held == 0
    for _ in range(17):
        step({0, 2})
        assert 20 - st.free_pages() == sum(-(-st.pos(s) // 8) for s in (0, 2))  # none for sequence 1
    step({2})
    step(set())
    assert st.pos(1) == 0
    st.prefill(t[100:117], 1)  # a new session in its place
    alone[1].reset()
    alone[1].prefill(t[100:117])
    for _ in range(4):
        step({0, 1, 2})
    step({1})
    ops.check_device_error()


def test_idle_sequences_need_nothing(model):
    """A full pool, and a sequence at its longest, hold up nobody else."""
    st = CudaState(model, 2, 128, paged=PagedConfig(17, 8))
    st.prefill(tokens(128, 1), 0)
    with pytest.raises(_lib.VtbError):
        st.step([4, 5])  # sequence 0 is full
    ref = CudaState(model, 1, 128)
    for tok in tokens(8, 2):
        (a, x), (b, y) = ref.step([tok]), st.step([-1, tok])
        assert near(b[1], a[0], LOGITS) and x[0] == y[1]
    assert st.free_pages() == 0 and st.pos(0) == 128
    with pytest.raises(_lib.VtbError) as e:
        st.step([-1, 9])  # no page for sequence 1
    assert e.value.status == -7 and st.pos(1) == 8
    st.step([-1, -1])
    ops.check_device_error()


def test_idle_is_for_steps_of_paged_states(model):
    paged, plain = CudaState(model, 2, 16, paged=PagedConfig(8, 16)), CudaState(model, 2, 16)
    for st, toks in ((plain, [-1, 4]), (paged, [-2, 4]), (paged, [SMALL.vocab_size, 4])):
        with pytest.raises(_lib.VtbError):
            st.step(toks)
        assert begin(st, toks) == -1
    with pytest.raises(_lib.VtbError):
        paged.prefill([3, -1, 4], 0)
    assert paged.pos(0) == 0 and paged.free_pages() == 8


def test_refused_calls_leave_a_begun_token(model):
    """A prefill that finds no page, or holds a bad token, changes nothing: the token that was begun goes on."""
    pc = PagedConfig(6, 16)
    st, want = CudaState(model, 2, 64, paged=pc), CudaState(model, 2, 64, paged=pc)
    t = tokens(60, 4)
    for s in (st, want):
        s.prefill(t[:20], 0)
        s.prefill(t[:33], 1)
    la, aa = want.step([7, 8], graph=False)
    assert begin(st, [7, 8]) == 0
    for bad in (t[:50], np.array([5, SMALL.vocab_size])):  # no page; no such token
        with pytest.raises(_lib.VtbError):
            st.prefill(bad, 0)
    for layer in range(SMALL.n_layers):
        assert st.lib.vtb_cuda_layer_step(st.h, layer) == 0
    assert st.lib.vtb_cuda_final_step(st.h) == 0
    logits, arg = np.empty((2, SMALL.vocab_size), np.float32), np.empty(2, np.int32)
    assert st.lib.vtb_cuda_finalize_token(st.h, logits.ctypes.data, arg.ctypes.data) == 0
    assert np.array_equal(logits, la) and np.array_equal(arg, aa)
    assert st.pos(0) == 21 and st.pos(1) == 34
    ops.check_device_error()


def test_prompt_over_a_token_that_was_given_up(tall):
    """Layers of a begun token are still queued when a prompt takes its place: they run on the rows and the table that
    they were queued with, so no page is missing."""
    n = 512
    pc = PagedConfig(n + 32, 8)
    st, want = CudaState(tall, n, n, paged=pc), CudaState(tall, 1, 128, paged=pc)
    t = np.random.default_rng(6).integers(3, TALL.vocab_size, 100)
    a, x = want.prefill(t)
    assert begin(st, [5] * n) == 0
    for _ in range(200):  # about 30 us each on the device, queued faster than that
        assert st.lib.vtb_cuda_final_step(st.h) == 0
    assert begin(st, [6] * n) == 0  # its rows are copied behind them
    for layer in range(TALL.n_layers):
        assert st.lib.vtb_cuda_layer_step(st.h, layer) == 0
    b, y = st.prefill(t)
    ops.check_device_error()
    assert near(b, a, LOGITS) and x == y
