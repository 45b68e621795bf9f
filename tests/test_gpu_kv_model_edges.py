"""Models over the paged cache's operators on a B200: what a call may depend on."""
import numpy as np
import pytest

from test_gpu_kv_model import _model

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd", [64, 128])
def test_a_prompt_does_not_depend_on_the_room(lrs, backend, hd):
    """The form of the attention goes by the positions in use, not by those that the slot
    has room for: the same bits at any max_seq_len, by prompt chunks and token by token."""
    prompt = lrs.prompt_tokens(5, 1088, 2000)  # whole chunks; the CTAs' parts differ between the forms
    got = []
    for room in (1152, 2048, 16384):
        _, _, m = _model(lrs, backend, "Q8_0", hd, seqs=1, max_seq=room)
        logits, _ = m.prefill(prompt)
        got.append([logits] + [m.forward_token(7 + i, 1088 + i)[0] for i in range(3)])
    for other in got[1:]:
        for a, b in zip(got[0], other):
            assert np.array_equal(a, b)
