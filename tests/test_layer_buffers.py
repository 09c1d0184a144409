"""What rope_append_paged takes as a compressed pool, checked without a GPU: sizes and types of the arrays
and words, which the kernel writes by address.

No counterpart in the reference (paged caches and the rotation on the way into them)."""
import pytest
import torch

from exactkv_amd import layer

H, D, PAGES = 2, 128, 4


def _pool():
    u8, i32 = torch.uint8, torch.int32
    shapes = dict(sm=((1, 16 * PAGES, H, D), u8), code=((1, 16 * PAGES, H, D // 2), u8), base=((1, PAGES, H, D), u8),
                  rowmask=((1, PAGES, H), i32), rowoff=((1, PAGES, H), i32), raw=((200, D), torch.bfloat16),
                  cnt=((1,), i32), before=((1,), i32), arrivals=((1,), i32))
    # 16-byte aligned whatever the host's allocator gives
    buf = {k: torch.zeros(torch.Size(s).numel() * t.itemsize + 64, dtype=u8) for k, (s, t) in shapes.items()}
    buf = {k: x[-x.data_ptr() % 16:][:torch.Size(shapes[k][0]).numel() * shapes[k][1].itemsize].view(shapes[k][1])
           .view(shapes[k][0]) for k, x in buf.items()}
    return dict(buf, cap=100, TS=16 * PAGES, H=H, D=D)


def test_a_sound_pool_is_taken():
    ptrs, cap, rows, pages = layer._pool_args(_pool(), H, D, -1, "kbuf")
    assert len(ptrs) == 9 and (cap, rows, pages) == (100, 200, PAGES)


@pytest.mark.parametrize("name,dtype", [("sm", torch.bool), ("sm", torch.int8), ("code", torch.int16), ("base", torch.float16),
                                        ("rowmask", torch.int16), ("rowmask", torch.int64), ("rowoff", torch.uint8),
                                        ("rowoff", torch.float32), ("raw", torch.uint8), ("raw", torch.float16),
                                        ("cnt", torch.int64), ("cnt", torch.uint8), ("before", torch.int16),
                                        ("arrivals", torch.int64), ("arrivals", torch.uint8)], ids=str)
def test_arrays_of_another_type_are_refused(name, dtype):
    buf = _pool()
    n = buf[name].numel()
    wide = torch.zeros(n * dtype.itemsize + 64, dtype=torch.uint8)
    buf[name] = wide[-wide.data_ptr() % 16:][:n * dtype.itemsize].view(dtype).view(buf[name].shape)
    with pytest.raises(ValueError, match="kbuf"):
        layer._pool_args(buf, H, D, -1, "kbuf")


@pytest.mark.parametrize("change", [dict(cnt=0), dict(before=0), dict(arrivals=0), dict(TS=60), dict(raw="flat"), dict(cap=-1)],
                         ids=str)
def test_words_and_sizes_that_do_not_fit_are_refused(change):
    buf = _pool()
    (name, to), = change.items()
    if to == 0:
        buf[name] = buf[name][:0]
    elif to == "flat":
        buf[name] = buf[name].view(-1, 8, D)
    else:
        buf[name] = to
    with pytest.raises(ValueError, match="kbuf"):
        layer._pool_args(buf, H, D, -1, "kbuf")
