"""Windowed attention, linear attention and the choice of a token on the GPU where their inputs are not ordinary: settings that are
no numbers, logits and states near the ends of f32, infinities and NaN under decays that vanish."""
import numpy as np
import pytest

from test_gpu_decoders import check_sample, f32, rng

pytestmark = pytest.mark.gpu

# ---- the choice of a token ----------------------------------------------------------------------------

FORMS = [65, 300, 5000, 30011]     # vocabularies of few rows: sorted by a wavefront, 256 threads, 1024 threads, several blocks a row


@pytest.mark.parametrize('V', FORMS)
@pytest.mark.parametrize('how', [dict(), dict(top_k=5), dict(top_p=0.9)], ids=['none', 'k', 'p'])
def test_sample_a_temperature_that_is_no_number_takes_the_largest_logit(V, how):
    r = rng(V, 101)
    heat = f32(np.where(np.arange(8) % 2, np.nan, 0.9))
    heat[6] = -1
    check_sample(f32(r.standard_normal((8, V))), f32(r.uniform(0.5, 1, 8)), temperature=heat, **how)
