"""Prompts longer than a state's rows: the chunks' rows share one staging buffer in pinned memory."""
import numpy as np
import pytest

from vantablack_b200 import synth as S
from vantablack_b200.model import Context, CudaModel, CudaState, HostWeights, LlamaConfig, PagedConfig

pytestmark = pytest.mark.gpu

TALL = LlamaConfig(dim=256, n_layers=2, n_heads=4, n_kv_heads=2, head_dim=64, ffn_dim=512, vocab_size=32768, max_seq=1600,
                   rope_base=10000.0)
LOGITS = 1e-3  # the bar of the forward loop against the oracle


@pytest.mark.parametrize("paged", [None, PagedConfig(700, 16, S.F32)])
def test_chunks_behind_queued_work(paged):
    """Milliseconds of work are queued before the prompt's first chunk, so its rows are still to be copied when the host
    comes to the second one."""
    n = 512
    m = CudaModel(Context(0), HostWeights(TALL, seed=7))
    st, want = CudaState(m, n, n, paged=paged), CudaState(m, 1, 1600, paged=paged)
    t = np.random.default_rng(4).integers(3, TALL.vocab_size, 1537)
    a, x = want.prefill(t)
    assert st.lib.vtb_cuda_begin_token(st.h, np.full(n, 5, np.int32).ctypes.data) == 0
    for _ in range(200):  # given up: about 30 us each on the device, queued faster than that
        assert st.lib.vtb_cuda_final_step(st.h) == 0
    b, y = st.prefill(t)
    assert np.abs(b - a).max() <= LOGITS * np.abs(a).max() and x == y
    m.close()
