"""Serving operators without a GPU: argument checks of the paged cache, and the oracle the GPU tests use."""
import math

import numpy as np
import pytest

import serve_oracle as so


def pages(pkg, **kw):
    a = dict(d_k=4096, d_v=8192, n_pages=10, n_kv=8, page_tokens=64, head_dim=128, type=pkg.KV_E4M3, d_k_scale=64, d_v_scale=128)
    a.update(kw)
    return pkg.KvPages(**a)


def test_cache_sizes_taken_and_declined(pkg):
    for P in (16, 32, 64, 128):
        for hd in (64, 96, 128, 192, 256):
            for ty in (pkg.KV_F16, pkg.KV_E4M3):
                assert pkg.kv_check(pages(pkg, page_tokens=P, head_dim=hd, type=ty), None, 32) == 1
    for kw in (dict(page_tokens=0), dict(page_tokens=8), dict(page_tokens=48), dict(page_tokens=256), dict(head_dim=0), dict(head_dim=80),
               dict(head_dim=512), dict(n_kv=0), dict(n_kv=65536)):
        assert pkg.kv_check(pages(pkg, **kw)) == 0, kw
    for heads, want in ((8, 1), (12, 0), (7, 0), (40, 1), (80000, 0)):
        assert pkg.kv_check(pages(pkg), None, heads) == want


def test_cache_argument_errors(pkg):
    packed = 8 * 64 * 128
    for kw in (dict(d_k=0), dict(d_v=0), dict(d_k=4104), dict(d_v=8), dict(n_pages=0), dict(type=2), dict(type=-1), dict(d_k_scale=0),
               dict(d_v_scale=0), dict(page_stride=packed - 16), dict(page_stride=packed + 8), dict(page_stride=1 << 40)):
        assert pkg.kv_check(pages(pkg, **kw)) == -1, kw
    assert pkg.kv_check(pages(pkg, type=pkg.KV_F16, d_k_scale=0, d_v_scale=0)) == 1
    assert pkg.kv_check(pages(pkg, type=pkg.KV_F16, page_stride=packed + 8)) == 1
    assert pkg.kv_check(pages(pkg, page_stride=3 * packed)) == 1
    assert pkg.kv_check(None) == -1


def test_batch_argument_errors(pkg):
    def batch(**kw):
        a = dict(n_seq=2, n_rows=5, d_row0=16, d_ctx=32, d_pages=64, pages_ld=4)
        a.update(kw)
        return pkg.KvBatch(**a)
    assert pkg.kv_check(pages(pkg), batch()) == 1
    assert pkg.kv_check(pages(pkg), batch(n_seq=0, d_row0=0, d_ctx=0, d_pages=0)) == 1
    assert pkg.kv_check(pages(pkg), batch(pages_ld=0, d_pages=0)) == 1
    for kw in (dict(d_row0=0), dict(d_ctx=0), dict(d_pages=0), dict(n_seq=1 << 24), dict(n_rows=1 << 31), dict(pages_ld=1 << 24)):
        assert pkg.kv_check(pages(pkg), batch(**kw)) == -1, kw


def test_calls_without_a_handle_fail(pkg):
    L = pkg.load_library()
    assert L.strix_cuda_kv_append_dev(None, pages(pkg), None, None, 0, None, 0, None, 0, None, 0, None, 0, None) == -1
    assert L.strix_cuda_attn_pages_dev(None, pages(pkg), None, 8, None, 0, 1.0, 0, None, 0, None, 0, None) == -1
    assert L.strix_cuda_attn_pages_workspace(None, pages(pkg), None, 8) == 0
    assert L.strix_cuda_sample_dev(None, None, 1, 1, 1, None, None, None, None, None) == -1
    assert L.strix_cuda_decode_step_sample(None, None, 0, 1.0, 0, 1.0, 0.0, 0.5, None, None) == -1


def test_oracle_e4m3_and_scale():
    v = so.e4m3_value(np.arange(127, dtype=np.uint8))
    assert v[0] == 0 and v[1] == 2.0 ** -9 and v[0x7e] == 448.0 and (np.diff(v) > 0).all()
    assert (so.e4m3_value(np.arange(128, 255, dtype=np.uint8)) == -v).all()
    for amax in (0.0, 1e-45, 1.0, 448.0, 448.1, 3.5, 1.75 * 2.0 ** 20, 1.76 * 2.0 ** 20, 3e38):
        s = so.scale_for(amax)
        assert math.frexp(s)[0] == 0.5 and amax <= 448 * s and (amax > 224 * s or s == 2.0 ** -120)


def test_oracle_rotation_keeps_pairs_and_relative_positions():
    rng = np.random.RandomState(0)
    q, k = rng.randn(1, 64), rng.randn(1, 64)
    for rope in (1, 2):
        dot = lambda a, b: float((so.prepared(q, None, a, rope, 1e4, 0, norm=False) * so.prepared(k, None, b, rope, 1e4, 0, norm=False)).sum())  # noqa: E731
        assert abs(dot(105, 100) - dot(5, 0)) < 1e-10
        assert abs((so.prepared(q, None, 77, rope, 1e4, 0, norm=False) ** 2).sum() - (q ** 2).sum()) < 1e-10


@pytest.mark.parametrize("kw,ids", [(dict(), {0, 1, 2, 3}), (dict(top_k=2), {1, 3}), (dict(top_p=0.5), {3}), (dict(min_p=0.2), {1, 3}), (dict(temperature=0.0), {3})])
def test_oracle_draw_keeps_the_right_tokens(kw, ids):
    x = np.log(np.array([0.1, 0.3, 0.05, 0.55]))
    assert {so.draw(x, (i + 0.5) / 200, **kw)[0] for i in range(200)} == ids
