"""The 4-bit key/value cache's calls refuse what they cannot do, before they look for a device (CPU)."""
import pytest

import zvdb_amd as zv

A = 0x10000  # an address that is aligned; nothing is read through it on the host


def layout(**kw):
    return zv.KVLayout(**{**dict(head_dim=64, kv_heads=2, page_size=16, pages=8), **kw})


def refused(call, code=1):
    with pytest.raises(zv.ZvdbError) as e:
        call()
    assert e.value.code == code, e.value
    assert len(str(e.value)) > 20


@pytest.mark.parametrize("bad", [dict(head_dim=0), dict(head_dim=4), dict(head_dim=60), dict(head_dim=264), dict(kv_heads=0), dict(kv_heads=1025),
                                 dict(page_size=0), dict(page_size=8), dict(page_size=24), dict(page_size=512), dict(pages=0), dict(pages=2**31)])
def test_layouts_that_are_refused(bad):
    refused(lambda: layout(**bad))


@pytest.mark.parametrize("d,w", [(8, 64), (64, 64), (72, 128), (128, 128), (136, 256), (256, 256)])
def test_page_bytes(d, w):
    assert layout(head_dim=d, kv_heads=3, page_size=32).page_bytes == 32 * 3 * (w + w // 16)


def plan(lay, lengths=A, new=A + 64, n=2, ring=A, ring_size=8, cursor=A, tables=A, stride=4, starts=A, slots=A, cap=8, out_lengths=A + 128,
         out_cursor=A + 64, status=A):
    lay.plan_dev(lengths, new, n, ring, ring_size, cursor, tables, stride, starts, slots, cap, out_lengths, out_cursor, status)


@pytest.mark.parametrize("bad", [dict(lengths=0), dict(new=0), dict(ring=0), dict(cursor=0), dict(tables=0), dict(starts=0), dict(slots=0),
                                 dict(out_lengths=0), dict(out_cursor=0), dict(status=0), dict(n=16385), dict(ring_size=0), dict(stride=0),
                                 dict(cap=2**31), dict(cursor=A + 4), dict(out_cursor=A + 4), dict(slots=A + 4), dict(out_cursor=A), dict(out_lengths=A)])
def test_plan_refuses(bad):
    refused(lambda: plan(layout(), **bad))


def append(lay, cache=A, k=A, ks=128, v=A, vs=128, type=1, n=3, slots=A):
    lay.append_dev(cache, k, ks, v, vs, type, n, slots)


@pytest.mark.parametrize("bad", [dict(cache=0), dict(k=0), dict(v=0), dict(slots=0), dict(type=2), dict(ks=120), dict(vs=120), dict(ks=132), dict(k=A + 8),
                                 dict(v=A + 8), dict(cache=A + 8), dict(slots=A + 4)])
def test_append_refuses(bad):
    refused(lambda: append(layout(), **bad))


@pytest.mark.parametrize("bad", [dict(cache=0), dict(slots=0), dict(type=7), dict(k=A + 8), dict(v=A + 8), dict(cache=A + 8), dict(slots=A + 4)])
def test_read_refuses(bad):
    a = {**dict(cache=A, slots=A, n=3, k=A, v=A, type=0), **bad}
    refused(lambda: layout().read_dev(a["cache"], a["slots"], a["n"], a["k"], a["v"], a["type"]))


def attend(lay, cache=A, q=A, q_stride=256, type=1, heads=4, n=2, starts=A, rows=2, max_new=1, lengths=A, tables=A, stride=4, max_length=64, scale=0.125,
           ws=A, ws_bytes=1 << 40, out=A, lse=A):
    lay.attend_dev(cache, q, q_stride, type, heads, n, starts, rows, max_new, lengths, tables, stride, max_length, scale, True, ws, ws_bytes, out, lse)


@pytest.mark.parametrize("bad", [dict(cache=0), dict(q=0), dict(starts=0), dict(lengths=0), dict(tables=0), dict(out=0), dict(q=A + 8), dict(out=A + 8),
                                 dict(cache=A + 8), dict(type=2), dict(heads=1), dict(heads=3), dict(heads=0), dict(q_stride=248), dict(q_stride=260),
                                 dict(stride=0), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(n=1 << 24),
                                 dict(rows=2**31), dict(max_length=2**31), dict(scale=3e38), dict(rows=2**30, max_new=2**30, heads=4)])
def test_attend_refuses(bad):
    refused(lambda: attend(layout(), **bad))


def selected(lay, cache=A, q=A, q_stride=256, type=1, heads=4, n=2, ids=A, counts=A, k=5, lengths=A, tables=A, stride=4, scale=0.125, out=A, lse=A):
    lay.attend_selected_dev(cache, q, q_stride, type, heads, n, ids, counts, k, lengths, tables, stride, scale, out, lse)


@pytest.mark.parametrize("bad", [dict(cache=0), dict(q=0), dict(ids=0), dict(lengths=0), dict(tables=0), dict(out=0), dict(ids=A + 4), dict(type=9), dict(heads=5),
                                 dict(q_stride=128), dict(stride=0), dict(scale=0.0), dict(k=2**31), dict(out=A + 4)])
def test_selected_refuses(bad):
    refused(lambda: selected(layout(), **bad))


@pytest.mark.parametrize("stride", [-128, -2**40, 2**40, 2**63, 2**64 - 8])
def test_strides_that_wrap_are_refused(stride):
    refused(lambda: append(layout(), ks=stride))
    refused(lambda: append(layout(), vs=stride))
    refused(lambda: attend(layout(), q_stride=stride))
    refused(lambda: selected(layout(), q_stride=stride))


def test_nothing_to_do_is_done_without_a_device():
    lay = layout()
    append(lay, n=0)
    lay.read_dev(A, A, 0, A, A, 0)
    lay.read_dev(A, A, 4, 0, 0, 0)
    attend(lay, n=0)
    attend(lay, rows=0)
    attend(lay, max_new=0)
    selected(lay, n=0)


def test_calls_without_a_device_say_so():
    if zv.device_count() > 0:
        pytest.skip("a GPU is visible")
    lay = layout()
    for call in (plan, append, attend, selected, lambda l: l.read_dev(A, A, 1, A, A, 0), lambda l: l.attend_workspace(1, 4, 2, 2, 1, 64)):
        refused(lambda: call(lay), 7)
