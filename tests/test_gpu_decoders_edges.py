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


@pytest.mark.parametrize('V', FORMS)
@pytest.mark.parametrize('temperature', [1e38, 2.0 ** 127, 3e38])
@pytest.mark.parametrize('how', [dict(), dict(top_k=50), dict(top_p=0.8), dict(min_p=0.1)], ids=['none', 'k', 'p', 'm'])
def test_sample_logits_whose_difference_passes_f32(V, temperature, how):
    """Each weighs by its distance to the largest, also where f32 cannot hold that."""
    r = rng(V, 102)
    logits, u = f32(3.4e38 * r.uniform(-1, 1, (8, V))), f32(r.random(8))
    logits[4:6] = np.where(r.random((2, V)) < 0.1, np.float32(2e38), np.float32(-2e38)) * f32(r.uniform(0.9, 1, (2, V)))
    logits[6, ::2] = -np.inf
    check_sample(logits, u, temperature=temperature, **how)


@pytest.mark.parametrize('V', FORMS)
def test_sample_limits_out_of_range_keep_the_first_or_all(V):
    """In tensors. The first of the order is always kept: alone by a min_p above 1 or not a number and by a top_p that is not above
    0, equal logits behind it or not; a min_p below 0 and a top_p that is 1 at least or not a number do not limit."""
    r = rng(V, 103)
    logits = f32(np.round(r.standard_normal((24, V))))       # many equal ones at the top
    p, m = np.ones(24, np.float32), np.zeros(24, np.float32)
    m[:4], m[4:8], m[8:10], m[10:12] = 3.0, np.nan, np.inf, np.nextafter(np.float32(1), np.float32(2))
    p[12:14], p[14:16], p[16:18], p[18:20], m[20:22], p[22:] = 0.0, -0.5, -np.inf, np.nan, -0.5, np.inf
    k = np.where(np.arange(24) % 2, 30, 0).astype(np.int32)
    got = check_sample(logits, f32(r.uniform(0.3, 1, 24)), top_p=p, min_p=m, top_k=k)
    alone = np.arange(24) < 18
    assert (got[alone] == logits[alone].argmax(1)).all() and (got[~alone] != logits[~alone].argmax(1)).any()
    check_sample(logits, f32(r.uniform(0.3, 1, 24)), min_p=m)
