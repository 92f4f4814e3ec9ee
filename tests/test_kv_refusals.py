"""What the cache, attention and draft entry points refuse, on the CPU: every refusal comes before any launch, with a reason."""

import ctypes

import pytest
import torch

import w4a16

CONFIG = w4a16.W4A16_ERR_CONFIG
A = 1 << 20  # addresses that nothing reads: a refused call launches nothing


def cache(**more):
    f = dict(k=A, v=A * 64, k_scale=None, v_scale=None, format=0, num_pages=4, page_size=16, kv_heads=2, head_dim=64)
    f.update(more)
    return w4a16._KvCacheStruct(**f)


def batch(**more):
    f = dict(page_table=A * 512, kv_lens=A * 513, starts=A * 514, seqs=2, rows=3, table_pages=2, table_stride=2, max_new=0, max_kv=0)
    f.update(more)
    return w4a16._KvBatchStruct(**f)


def write(c=None, b=None, k=A * 256, v=A * 320, ks=(128, 64), vs=(128, 64)):
    c, b = c or cache(), b or batch()
    return w4a16.lib.w4a16_kv_write_bf16(ctypes.byref(c), ctypes.byref(b), k, *ks, v, *vs, None)


def read(c=None, b=None, k=A * 256, v=A * 320):
    c, b = c or cache(), b or batch()
    return w4a16.lib.w4a16_kv_read_bf16(ctypes.byref(c), ctypes.byref(b), k, v, None)


def attend(c=None, b=None, q=A * 256, qs=(256, 64), heads=4, scale=0.125, window=0, out=A * 320, os=(256, 64), lse=None,
           ws=A * 1024, ws_bytes=1 << 28):
    c, b = c or cache(), b or batch()
    return w4a16.lib.w4a16_paged_attention_bf16(ctypes.byref(c), ctypes.byref(b), q, *qs, heads, scale, 1, window, out, *os, lse,
                                                ws, ws_bytes, None)


def verify(target=A * 256, ts=(400000, 100000), draft=A * 320, ds=(300000, 100000), tokens_in=A, lens=None, uniforms=A * 2, accepted=A * 3,
           tokens=A * 4, seqs=2, steps=3, vocab=100000, ws=A * 5, ws_bytes=1 << 20):
    return w4a16.lib.w4a16_verify_drafts_f32(target, *ts, draft, *ds, tokens_in, lens, uniforms, accepted, tokens, seqs, steps,
                                             vocab, ws, ws_bytes, None)


@pytest.mark.parametrize("fields,why", [
    (dict(format=3), "W4A16_KV"), (dict(head_dim=96), "head_dim"), (dict(head_dim=0), "head_dim"),
    (dict(page_size=12), "power of two"), (dict(page_size=4), "power of two"), (dict(page_size=131072), "power of two"),
    (dict(kv_heads=0), "extents"), (dict(num_pages=0), "extents"), (dict(num_pages=1 << 27), "extents"),
    (dict(k=None), "null"), (dict(v=None), "null"), (dict(k=A + 8), "aligned"), (dict(format=1), "scales"),
    (dict(format=2, k_scale=A * 3), "scales"), (dict(format=2, k_scale=A * 3 + 4, v_scale=A * 4), "aligned"),
])
def test_caches(fields, why):
    for call in (write, read, attend):
        assert call(c=cache(**fields)) == CONFIG
        assert why in w4a16.last_error()


@pytest.mark.parametrize("fields,why", [
    (dict(seqs=-1), "extents"), (dict(rows=-1), "extents"), (dict(rows=(1 << 25) + 1), "extents"), (dict(table_pages=-1), "extents"),
    (dict(table_stride=1), "extents"), (dict(max_new=-1), "extents"), (dict(max_kv=-5), "extents"), (dict(kv_lens=None), "null"),
    (dict(starts=None), "null"), (dict(page_table=None), "null"), (dict(starts=A + 2), "aligned"),
])
def test_batches(fields, why):
    for call in (write, read, attend):
        assert call(b=batch(**fields)) == CONFIG
        assert why in w4a16.last_error()


@pytest.mark.parametrize("call,args,why", [
    (write, dict(k=None), "null"), (write, dict(v=A * 320 + 8), "aligned"), (write, dict(ks=(130, 64)), "strides"),
    (write, dict(vs=(128, -64)), "strides"), (write, dict(ks=(1 << 62, 64)), "strides"), (write, dict(k=A + 64), "overlap"),
    (write, dict(c=cache(v=A + 1024)), "overlap"), (write, dict(c=cache(format=1, k_scale=A * 256, v_scale=A * 3)), "scales"),
    (read, dict(v=None), "null"), (read, dict(k=A * 256 + 2), "aligned"), (read, dict(v=A * 256 + 64), "overlap"),
    (read, dict(k=A * 64), "overlap"), (read, dict(c=cache(format=2, k_scale=A * 256, v_scale=A * 3)), "overlap"),
    (attend, dict(heads=3), "multiple"), (attend, dict(heads=0), "multiple"), (attend, dict(heads=1 << 30), "multiple"),
    (attend, dict(scale=float("nan")), "scale"), (attend, dict(scale=float("inf")), "scale"), (attend, dict(window=-1), "window"),
    (attend, dict(q=None), "null"), (attend, dict(out=None), "null"), (attend, dict(out=A * 320 + 8), "aligned"),
    (attend, dict(lse=A * 400 + 2), "aligned"), (attend, dict(qs=(256, 4)), "strides"), (attend, dict(os=(-256, 64)), "strides"),
    (attend, dict(os=(256, 32)), "each other"), (attend, dict(os=(192, 64)), "each other"), (attend, dict(os=(0, 64)), "each other"),
    (attend, dict(out=A * 256 + 128), "overlap"), (attend, dict(out=A), "overlap"), (attend, dict(lse=A * 320), "overlap"),
    (attend, dict(lse=A * 256), "overlap"),
    (attend, dict(b=batch(max_kv=100000), ws=None), "workspace"), (attend, dict(b=batch(max_kv=100000), ws_bytes=64), "workspace"),
    (attend, dict(b=batch(max_kv=100000), ws=A * 256), "overlap"), (attend, dict(b=batch(max_kv=100000), ws=A * 64), "overlap"),
    (verify, dict(seqs=-1), "extents"), (verify, dict(seqs=65536), "extents"), (verify, dict(steps=-1), "extents"),
    (verify, dict(vocab=0), "extents"), (verify, dict(vocab=(1 << 28) + 1), "extents"), (verify, dict(target=None), "null"),
    (verify, dict(tokens_in=None), "null"), (verify, dict(uniforms=None), "null"), (verify, dict(accepted=None), "null"),
    (verify, dict(tokens=None), "null"), (verify, dict(ws=None), "null"), (verify, dict(draft=A * 320 + 2), "aligned"),
    (verify, dict(ws=A * 5 + 8), "aligned"), (verify, dict(ws_bytes=16), "workspace"), (verify, dict(ts=(-1, 100000)), "stride"),
    (verify, dict(accepted=A * 256), "overlap"), (verify, dict(tokens=A), "overlap"), (verify, dict(tokens=A * 3), "overlap"),
    (verify, dict(ws=A * 4), "overlap"),
])
def test_calls(call, args, why):
    assert call(**args) == CONFIG
    assert why in w4a16.last_error()


def test_nothing_to_do():
    for b in (batch(rows=0), batch(seqs=0), batch(seqs=0, kv_lens=None, starts=None, page_table=None)):
        assert write(b=b) == 0 and read(b=b) == 0 and attend(b=b) == 0
    assert verify(seqs=0) == 0


def test_workspaces():
    need = ctypes.c_size_t(7)
    one = cache(num_pages=1 << 20)
    lib = w4a16.lib
    sizes = []
    for most in (100, 2000, 50000):
        assert lib.w4a16_paged_attention_workspace(ctypes.byref(one), ctypes.byref(batch(max_kv=most)), 4, ctypes.byref(need)) == 0
        sizes.append(need.value)
    assert 0 == sizes[0] < sizes[1] < sizes[2]  # short sequences are not cut
    # many rows in many tiles: nothing to join
    many = batch(rows=1 << 16, seqs=1, max_new=1 << 16)
    assert lib.w4a16_paged_attention_workspace(ctypes.byref(one), ctypes.byref(many), 4, ctypes.byref(need)) == 0
    assert need.value == 0
    assert lib.w4a16_paged_attention_workspace(ctypes.byref(one), ctypes.byref(batch()), 4, None) == CONFIG
    assert lib.w4a16_paged_attention_workspace(None, ctypes.byref(batch()), 4, ctypes.byref(need)) == CONFIG
    assert lib.w4a16_verify_drafts_workspace(3, 2, 100000, ctypes.byref(need)) == 0 and need.value >= 3 * 16
    assert lib.w4a16_verify_drafts_workspace(3, 2, 1000, ctypes.byref(need)) == 0 and need.value == 0
    assert lib.w4a16_verify_drafts_workspace(3, 2, 100, None) == CONFIG


def test_binding():
    """The binding's own checks: tensors of the host, of other types and shapes."""
    host = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    for make in (lambda: w4a16.KvCache(host, host), lambda: w4a16.KvCache(host.float(), host.float()),
                 lambda: w4a16.KvCache(host, host[:2]), lambda: w4a16.KvCache(host.to(torch.int8), host.to(torch.int8)),
                 lambda: w4a16.KvCache.empty(4, 16, 2, 64, "fp4", device="cpu"),
                 lambda: w4a16.KvBatch(torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32),
                                       torch.zeros(2, dtype=torch.int32), 1),
                 lambda: w4a16.verify_drafts(torch.zeros(1, 2, 5), torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, 2))):
        with pytest.raises(w4a16.W4A16Error):
            make()
