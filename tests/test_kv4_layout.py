"""The 4-bit cache on the CPU: its layout restated twice, and what the entry points refuse before anything is launched."""
import pytest
import torch

import kv4_plain as plain
from glassbox_b200 import kernels


@pytest.mark.parametrize("hd", [32, 64, 96, 128, 256])
def test_every_channel_has_a_nibble_of_its_own(hd):
    for per in (8, 4):
        assert sorted(plain.nibble(c, hd, per) for c in range(hd)) == list(range(hd))


@pytest.mark.parametrize("hd, page_size", [(32, 16), (96, 48), (128, 32)])
def test_tokens_are_read_back_from_a_page(hd, page_size):
    (k, v), dense = plain.random_pool(2, 3, page_size, hd, 5)
    assert k.shape[-1] == kernels.kv4_page_bytes(page_size, hd)
    for pool, want, per in ((k, dense[0], 8), (v, dense[1], 4)):
        for off in (0, 15, page_size - 1):
            got = plain.numbers(*plain.read_token(pool[1, 2], off, hd, per))
            assert torch.equal(got, want[1, 2, off])
            page = torch.zeros_like(pool[1, 2])
            plain.write_token(page, off, *plain.read_token(pool[1, 2], off, hd, per), per)
            assert torch.equal(plain.numbers(*plain.read_token(page, off, hd, per)), want[1, 2, off])


def test_held_numbers_are_near_and_exact_in_bfloat16():
    x = torch.randn(50, 64, generator=torch.Generator().manual_seed(1), dtype=torch.float64)
    codes, scales = plain.hold(x)
    got = plain.numbers(codes, scales)
    assert torch.equal(got.to(torch.bfloat16).double(), got)
    d = scales.abs().repeat_interleave(32, dim=-1)
    clipped = (x / scales.repeat_interleave(32, dim=-1)) > 7.5
    assert ((got - x).abs() <= d * torch.where(clipped, 1.01 + 8 / 32, 0.5 + 8 / 32 / 8)).all()


def _operands(n=3, nh=4, nkv=2, hd=64, page_size=16, pages=5, dtype=torch.bfloat16):
    size = kernels.kv4_page_bytes(page_size, hd)
    return dict(qkv=torch.zeros(n, (nh + 2 * nkv) * hd, dtype=dtype), q=torch.zeros(n, nh * hd, dtype=dtype), cos_sin=torch.zeros(9, hd // 2, 2),
                positions=torch.zeros(n, dtype=torch.int32), slots=torch.zeros(n, dtype=torch.int32),
                kcache=torch.zeros(pages, nkv, size, dtype=torch.uint8), vcache=torch.zeros(pages, nkv, size, dtype=torch.uint8), nh=nh, nkv=nkv, hd=hd,
                rot=hd, page_size=page_size, write_kv=True, status=torch.zeros(1, dtype=torch.int32))


BAD_WRITES = [dict(hd=48, rot=48), dict(page_size=24), dict(q=torch.zeros(3, 255, dtype=torch.bfloat16)), dict(q=torch.zeros(3, 256)),
              dict(rot=66), dict(rot=31), dict(cos_sin=torch.zeros(9, 31, 2)), dict(cos_sin=torch.zeros(9, 32, 2, dtype=torch.float64)),
              dict(positions=torch.zeros(2, dtype=torch.int32)), dict(slots=torch.zeros(3, dtype=torch.int64)), dict(kcache=torch.zeros(5, 2, 575, dtype=torch.uint8)),
              dict(vcache=torch.zeros(4, 2, 576, dtype=torch.uint8)), dict(kcache=torch.zeros(5, 2, 576, dtype=torch.int8)),
              dict(qkv=torch.zeros(3, 500, dtype=torch.bfloat16)), dict(qkv=torch.zeros(1, 512, dtype=torch.bfloat16).expand(3, 512)), dict(hd=288, rot=0)]


@pytest.mark.parametrize("change", BAD_WRITES, ids=[str(i) for i in range(len(BAD_WRITES))])
def test_refused_writes(change):
    with pytest.raises(kernels.KernelError):
        kernels.kv4_write(**{**_operands(), **change})


def test_there_is_no_cpu_path():
    with pytest.raises(kernels.KernelError, match="CUDA"):
        kernels.kv4_write(**_operands())
    with pytest.raises(kernels.KernelError, match="CUDA"):
        kernels.token_logprobs(torch.zeros(2, 9), torch.zeros(2, dtype=torch.int32), torch.zeros(2))


def _attention(n=3, nh=4, nkv=2, hd=64, page_size=16, pages=5, dtype=torch.bfloat16):
    o = _operands(n, nh, nkv, hd, page_size, pages, dtype)
    return dict(q=o["q"], out=torch.zeros_like(o["q"]), kcache=o["kcache"], vcache=o["vcache"], block_tables=torch.zeros(n, 4, dtype=torch.int32),
                row_seq=torch.zeros(n, dtype=torch.int32), positions=o["positions"], nh=nh, nkv=nkv, hd=hd, page_size=page_size, scale=0.1, window=None,
                max_context=64, parts=None, status=o["status"])


BAD_ATTENTION = [dict(nh=5), dict(out=torch.zeros(3, 256)), dict(q=torch.zeros(2, 256, dtype=torch.bfloat16)), dict(block_tables=torch.zeros(3, 4)),
                 dict(block_tables=torch.zeros(4, 3, dtype=torch.int32).t()), dict(row_seq=torch.zeros(2, dtype=torch.int32)), dict(page_size=20),
                 dict(out=torch.zeros(1, 256, dtype=torch.bfloat16).expand(3, 256)), dict(q=torch.zeros(3, 256, dtype=torch.float16), out=torch.zeros(3, 256, dtype=torch.float16))]


@pytest.mark.parametrize("change", BAD_ATTENTION, ids=[str(i) for i in range(len(BAD_ATTENTION))])
def test_refused_attention(change):
    with pytest.raises(kernels.KernelError):
        kernels.kv4_attention_decode(**{**_attention(), **change})


def test_refused_reads_and_pages_to_unpack_into():
    o = _operands()
    k = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    for bad in (dict(k=k[:, :, :32]), dict(v=k.float()), dict(slots=torch.zeros(2, dtype=torch.int32)), dict(page_size=32)):
        args = dict(kcache=o["kcache"], vcache=o["vcache"], slots=o["slots"], k=k, v=k.clone(), page_size=16, status=o["status"])
        with pytest.raises(kernels.KernelError):
            kernels.kv4_read(**{**args, **bad})
    pages = torch.zeros(5, 2, 16, 64, dtype=torch.bfloat16)
    args = dict(kcache=o["kcache"], vcache=o["vcache"], kpages=pages, vpages=pages.clone(), block_tables=torch.zeros(2, 4, dtype=torch.int32),
                seq_first_row=torch.zeros(3, dtype=torch.int32), seq_start_pos=torch.zeros(2, dtype=torch.int32), max_context=64, window=None,
                status=o["status"])
    for bad in (dict(kpages=pages[:4], vpages=pages[:4]), dict(vpages=pages.float()), dict(seq_first_row=torch.zeros(2, dtype=torch.int32)),
                dict(kpages=pages.transpose(1, 2), vpages=pages.transpose(1, 2))):
        with pytest.raises(kernels.KernelError):
            kernels.kv4_expand(**{**args, **bad})


def test_refused_scores():
    x, t, lp, i = torch.zeros(2, 40), torch.zeros(2, dtype=torch.int32), torch.zeros(2), torch.zeros(2, 4, dtype=torch.int32)
    for args in ((x.t(), t, lp), (x, t.long(), lp), (x, t[:1], lp), (x, t, lp[:1]), (x, t, lp, torch.zeros(3)), (x, t, lp, None, torch.zeros(2, 4), None),
                 (x, t, lp, None, torch.zeros(2, 3), i), (x, t, lp, None, None, i.long()), (x, t, lp, None, None, torch.zeros(2, 33, dtype=torch.int32)),
                 (x[:, :3], t, lp, None, None, i), (x, t, lp, None, None, i[:, :0])):
        with pytest.raises(kernels.KernelError):
            kernels.token_logprobs(*args)


@pytest.mark.parametrize("scale", [0.0, -0.1, float("nan"), float("inf")])
def test_refused_scales(scale):
    with pytest.raises(kernels.KernelError, match="positive"):
        kernels.kv4_attention_decode(**{**_attention(), "scale": scale})
