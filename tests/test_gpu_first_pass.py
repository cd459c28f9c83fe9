"""What a model clears on its first passes (row descriptors, merge counters) is cleared before they
use it, also while the default stream, which the model's stream does not wait for, is busy: a clear
that ran there once came after the upload of the rows and left a pass without them."""
import numpy as np
import pytest

from yue2_rs_b200 import Model, synth

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [20, 6, 2])
def test_first_passes_beside_a_busy_default_stream(rows):
    import torch
    c = synth.config_c1()
    c.vocab_size = 4096
    prompts = [[(37 * r + 11 * i) % 4096 for i in range(9 + r % 5)] for r in range(rows)]

    def run(busy):
        m = Model.synthetic(c, seed=5, std=0.02, norm_mean=1.0)
        try:
            caches = [m.new_cache(len(p) + 41) for p in prompts]
            out = [np.stack([m.forward(p, k) for p, k in zip(prompts, caches)])]
            if busy:
                torch.cuda._sleep(10_000_000)  # a few milliseconds: it ends while the passes below run
            for step in range(40):
                out.append(m.forward_rows(caches, [(7 * step + r) % 4096 for r in range(rows)]))
            return np.stack(out)
        finally:
            torch.cuda.synchronize()
            m.close()

    want = run(False)
    assert np.array_equal(run(True), want)
