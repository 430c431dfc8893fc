"""CPU tests of the cache operators' refusals at the edges of what their header allows (no device
needed: every refusal here happens before the library touches one)."""
import ctypes as C

import pytest

from test_cache_ops_cpu import INVALID, P, tree


@pytest.mark.parametrize("stride,cols", [(64, 0), (64, -1), (64, 65), (0, 0)])
def test_rows_of_weights_hold_their_columns(ckl, stride, cols):
    L = ckl.lib()
    assert L.ckl_cache_weights_ex(C.byref(tree(ckl)), P, P, stride, cols, 1.0, None) == INVALID
    assert L.ckl_cache_select_ex(P, stride, cols, P, P, 2, 8, 0, 0, P, P, None) == INVALID
    assert L.ckl_cache_compact_ex(P, 0x100000, P, P, P, 2, 2, 4, P, 8, P, None, P, stride, cols, None,
                                  None) == INVALID


def test_compact_refuses_what_it_would_write_under_its_readers(ckl):
    """The parts of one call read the lists and the page table while others write the caches, the
    weights and the lengths."""
    L = ckl.lib()
    # caches of 4 pages x 16 x 2 heads x 256 bytes = 32 KB; five sequences, lists of eight
    base = dict(k=0x100000, v=0x200000, indptr=0x1000, ind=0x2000, last=0x3000, idx=0x4000, cnt=0x5000, start=0x6000,
                acc=0x7000, new=0x8000)

    def call(**kw):
        f = {**base, **kw}
        return L.ckl_cache_compact_ex(f["k"], f["v"], f["indptr"], f["ind"], f["last"], 5, 2, 4, f["idx"], 8, f["cnt"],
                                      f["start"], f["acc"], 16, 10, f["new"], None)

    for new in (0x4000 - 16, 0x4000, 0x4000 + 32 * 4, 0x4000 + 39 * 4, 0x2000, 0x1000 + 20, 0x7000 + 72 * 4,
                0x100000 + 32764, 0x200000):
        assert call(new=new) == INVALID, hex(new)
    for acc in (0x4000 - 73 * 4, 0x4000 + 156, 0x2000, 0x1000, 0x3000, 0x5000, 0x6000, 0x100000, 0x200000 + 32764):
        assert call(acc=acc) == INVALID, hex(acc)
    for idx in (0x100000, 0x200000 - 156):
        assert call(idx=idx) == INVALID, hex(idx)


class Stream:
    cuda_stream = 0

    def __init__(self, dev):
        self.device_index = dev


@pytest.mark.parametrize("current,stream", [(1, None), (1, Stream(0)), (1, Stream(1)), (0, Stream(1))])
def test_params_of_another_device_are_refused(ckl, monkeypatch, current, stream):
    """Parameters made on cuda:0 and called while cuda:1 is current, or for a stream of cuda:1:
    refused before anything is launched or allocated. (Empty batches: nothing would run.)"""
    monkeypatch.setattr(ckl, "_raw_device", lambda: current)
    monkeypatch.setattr(ckl, "_raw_stream", lambda dev: 0)
    ap, tp = ckl.AppendParams(Hkv=1), ckl.TreeParams(Hq=1, Hkv=1)
    ap._dev = tp._dev = 0
    ap.q_rotated, ap._made, tp._keep = None, False, (None,)
    for call in (lambda: ckl.rope_append(ap, stream=stream), lambda: ckl.tree_attention(tp, stream=stream),
                 lambda: ckl.cache_weights(tp, None, None, stream=stream)):
        with pytest.raises(ckl.CklError, match="cuda:1") as e:
            call()
        assert e.value.status == INVALID


def test_rope_append_keeps_its_own_output_for_the_stream(ckl, monkeypatch):
    """q_out that make_append_params allocated, on the stream of its time, is written on the call's
    stream: its memory waits for that one. The caller's own q_out is the caller's."""
    monkeypatch.setattr(ckl, "_raw_device", lambda: 0)
    monkeypatch.setattr(ckl, "_raw_stream", lambda dev: 0)
    seen = []

    class Out:
        def record_stream(self, stream):
            seen.append(stream)

    p, s = ckl.AppendParams(Hkv=1), Stream(0)
    p._dev, p.q_rotated = 0, Out()
    for made, stream, want in ((False, s, []), (True, None, []), (True, s, [s])):
        p._made = made
        assert ckl.rope_append(p, stream=stream) is p.q_rotated and seen == want


def test_tree_mask_refuses_outputs_over_inputs(ckl):
    """5 tokens of 2 sequences, 2 words a row: masks of 40 bytes, positions of 20."""
    call = lambda mask=0x5000, pos=0x6000: ckl.lib().ckl_tree_mask(0x1000, 0x2000, 0x3000, 0x4000, 2, 5, 2, mask, pos, None)
    for pos in (0x1000 - 16, 0x1000, 0x1000 + 16, 0x2000 + 8, 0x3000, 0x4000 + 4, 0x5000 + 36, 0x5000 - 16):
        assert call(pos=pos) == INVALID, hex(pos)
    for mask in (0x1000 - 36, 0x1000 + 16, 0x2000 + 8, 0x3000, 0x4000):
        assert call(mask=mask) == INVALID, hex(mask)
