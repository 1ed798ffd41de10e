"""What the paged calls and vb_logits_process refuse: decided from the arguments
alone, before anything of CUDA is touched (the addresses here belong to nothing,
and no device is needed)."""
import ctypes as C

import pytest

import vb200

A = 1 << 20  # a 16-byte aligned address that is never followed


def cache(**k):
    c = dict(k=A, v=2 * A, dtype=0, num_pages=10, page_size=16, kv_heads=2, head_dim=128, stride_page=16 * 2 * 128,
             stride_pos=2 * 128, stride_head=128)
    c.update(k)
    return vb200.VBPagedCache(**c)


def batch(**k):
    b = dict(batch=2, tokens=5, max_new=4, max_len=64, q_start=A, lens=A, table=A, table_stride=4, status=None)
    b.update(k)
    return vb200.VBPagedBatch(**b)


def append(c=None, b=None, rope=None, io=0, heads=4, q=A, qo=A, k=A, v=A, q_row=512, q_head=128, qo_row=512, k_row=256):
    c, b = c or cache(), b or batch()
    return vb200.lib().vb_paged_append(C.addressof(c), C.addressof(b), C.addressof(rope) if rope else None, io, heads, q,
                                       q_row, q_head, qo, qo_row, q_head, k, k_row, 128, v, 256, 128, None)


def attn(c=None, b=None, io=0, heads=4, q=A, out=A, window=0, ws=A, ws_bytes=1 << 30, q_row=512, lse=None):
    c, b = c or cache(), b or batch()
    return vb200.lib().vb_paged_attn(C.addressof(c), C.addressof(b), io, heads, q, q_row, 128, out, 512, 128, lse, 0.1,
                                     window, ws, ws_bytes, None)


BAD_CACHE = [
    (dict(k=None), -1), (dict(v=None), -1), (dict(dtype=3), -1), (dict(dtype=1), -9), (dict(head_dim=96), -9),
    (dict(num_pages=0), -1), (dict(page_size=0), -1), (dict(kv_heads=0), -1), (dict(kv_heads=3), -1),
    (dict(stride_page=-4096), -1), (dict(stride_pos=257), -9), (dict(stride_head=130), -9), (dict(k=A + 4), -9),
    (dict(v=A + 8), -9), (dict(page_size=8), -1),  # the table's 4 pages hold 32 positions, max_len is 64
]
BAD_BATCH = [(dict(batch=-1), -1), (dict(tokens=-1), -1), (dict(max_new=-1), -1), (dict(max_len=-1), -1),
             (dict(table_stride=-1), -1), (dict(max_len=65), -1), (dict(q_start=None), -1), (dict(lens=None), -1),
             (dict(table=None), -1)]


@pytest.mark.parametrize("call", [append, attn])
@pytest.mark.parametrize("change,code", BAD_CACHE)
def test_bad_caches(call, change, code):
    assert call(c=cache(**change)) == code
    assert vb200.lib().vb_last_error()


@pytest.mark.parametrize("call", [append, attn])
@pytest.mark.parametrize("change,code", BAD_BATCH)
def test_bad_batches(call, change, code):
    assert call(b=batch(**change)) == code


@pytest.mark.parametrize("call", [append, attn])
def test_null_descriptors(call):
    L = vb200.lib()
    b = batch()
    assert L.vb_paged_attn(None, C.addressof(b), 0, 4, A, 512, 128, A, 512, 128, None, 0.1, 0, A, 1 << 30, None) == -1
    assert L.vb_paged_append(None, C.addressof(b), None, 0, 4, A, 512, 128, A, 512, 128, A, 256, 128, A, 256, 128,
                             None) == -1
    assert L.vb_paged_attn_workspace_bytes(None, C.addressof(b), 4) == 0


@pytest.mark.parametrize("call", [append, attn])
def test_types_that_do_not_go_together(call):
    assert call(io=7) == -1
    assert call(io=2) == -9            # 16-bit rows over an f32 cache
    assert call(c=cache(dtype=1)) == -9  # f32 rows over an f16 cache
    assert call(heads=3) == -1


def test_append_arguments():
    assert append(q=None) == -1 and append(qo=None) == -1
    assert append(k=None) == -1 and append(v=None) == -1
    assert append(q=A + 8, qo=A + 8) == -9 and append(k_row=258) == -9
    assert append(qo_row=1024) == -1  # in place with other strides
    rope = dict(cos_tab=A, sin_tab=A, rope_positions=64, rot=128, interleaved=0, q_norm=None, k_norm=None, eps=1e-6)
    for change, code in [(dict(rot=24), -9), (dict(rot=144), -9), (dict(rot=-16), -9), (dict(cos_tab=None), -1),
                         (dict(sin_tab=A + 4), -9), (dict(rope_positions=63), -5), (dict(q_norm=A + 4), -9)]:
        assert append(rope=vb200.VBPagedRope(**dict(rope, **change))) == code, change


def test_attn_arguments():
    assert attn(q=None) == -1 and attn(out=None) == -1
    assert attn(q=A + 4) == -9 and attn(q_row=514) == -9
    assert attn(window=-1) == -1
    c, b = cache(), batch(max_len=1024, table_stride=64)
    need = vb200.lib().vb_paged_attn_workspace_bytes(C.addressof(c), C.addressof(b), 4)
    assert need > 0
    assert attn(b=b, ws_bytes=need - 1) == -1 and attn(b=b, ws=None) == -1 and attn(b=b, ws=A + 8) == -9


def test_nothing_to_do_is_fine():
    for b in (batch(batch=0), batch(tokens=0), batch(batch=0, tokens=0, q_start=None, lens=None, table=None)):
        assert append(b=b) == 0 and attn(b=b) == 0
    assert vb200.lib().vb_paged_attn_workspace_bytes(C.addressof(cache()), C.addressof(batch(tokens=0)), 4) == 0


@pytest.mark.parametrize("heads,kv_heads,max_new,max_len,B", [(16, 8, 1, 4096, 4), (32, 4, 7, 100000, 1)])
def test_the_workspace_is_asked_for_alike_for_any_window(heads, kv_heads, max_new, max_len, B):
    c = cache(kv_heads=kv_heads, stride_pos=kv_heads * 128, stride_page=kv_heads * 128 * 16)
    b = batch(batch=B, tokens=B * max_new, max_new=max_new, max_len=max_len, table_stride=max_len // 16 + 1)
    need = vb200.lib().vb_paged_attn_workspace_bytes(C.addressof(c), C.addressof(b), heads)
    assert need > 0
    for w in (0, 1, 63, 64, 577, 4096):
        assert attn(c=c, b=b, heads=heads, window=w, ws_bytes=need - 1) == -1


def logits(p=A, out=A, dtype=0, rows=2, vocab=100, s_in=100, s_out=100, **rules):
    r = vb200.VBLogitsRules(**rules)
    return vb200.lib().vb_logits_process(p, s_in, out, s_out, dtype, rows, vocab, C.addressof(r), None)


def test_logits_arguments():
    assert logits(dtype=5) == -1 and logits(rows=-1) == -1 and logits(vocab=0) == -1
    assert logits(vocab=1 << 31, s_in=1 << 31, s_out=1 << 31) == -9
    assert logits(p=None) == -1 and logits(out=None) == -1
    assert logits(s_in=99) == -1 and logits(s_out=99) == -1 and logits(s_in=101) == -1
    assert logits(repetition=A) == -1 and logits(presence=A) == -1  # no history
    assert logits(hist_start=A, hist_total=-1) == -1 and logits(hist_start=A, hist_total=4) == -1
    assert logits(bias_start=A, bias_total=4, bias_ids=A) == -1
    assert logits(mask=A, mask_stride=3) == -1
    assert logits(rows=0) == 0
    assert vb200.lib().vb_logits_process(A, 100, A, 100, 0, 2, 100, None, None) == -1


def test_attention_does_not_run_in_place():
    # a row with an infinity or NaN in it is taken again from its q
    assert attn(q=A, out=A) == -1
    assert b"place" in vb200.lib().vb_last_error()


def test_addresses_that_do_not_fit_their_elements():
    # refused here: on the device an access at such an address is a fault
    for n in ("q_start", "lens", "table", "status"):
        assert attn(b=batch(**{n: A + 2})) == -9 and append(b=batch(**{n: A + 1})) == -9, n
    assert attn(lse=A + 2) == -9
    for dtype, off in ((0, 2), (0, 1), (1, 1), (2, 1)):
        assert logits(dtype=dtype, p=A + off) == -9 and logits(dtype=dtype, out=2 * A + off) == -9
    lists = dict(hist_start=A, hist_ids=A, hist_total=4, prompt_len=A, repetition=A, frequency=A, presence=A, bias_start=A,
                 bias_ids=A, bias_vals=A, bias_total=4, mask=A, mask_stride=4)
    for n, v in lists.items():
        if v == A:
            assert logits(**dict(lists, **{n: A + 2})) == -9, n


def test_positions_stay_far_from_32_bits():
    # tiles of keys are counted past the last position
    b = batch(max_len=(1 << 30) + 1, table_stride=1 << 30)
    assert attn(b=b) == -9 and b"keys" in vb200.lib().vb_last_error()
    assert attn(b=batch(max_len=0x7fffffff, table_stride=1 << 30)) == -9


def test_python_faces_refuse_what_is_not_on_the_device():
    torch = pytest.importorskip("torch")
    k = torch.zeros(4, 16, 2, 128)
    with pytest.raises(vb200.VBError):
        vb200.PagedCache(k, k.clone())
    with pytest.raises(vb200.VBError):
        vb200.PagedCache(k, k.clone().half())
    i = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(vb200.VBError):
        vb200.PagedBatch(i, i[:2], torch.zeros(2, 4, dtype=torch.int32), max_new=1, max_len=1, tokens=2)
    with pytest.raises(vb200.VBError):
        vb200.LogitsRules(prompt_len=i)
    x = torch.zeros(2, 10)
    with pytest.raises(vb200.VBError):
        vb200.logits_process(x, x, vb200.LogitsRules())
