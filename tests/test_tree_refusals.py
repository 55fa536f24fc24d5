"""What the operators of drafted tokens refuse, before anything is launched."""
import pytest
import torch

from glassbox_b200 import kernels

INT = torch.int32


def attention_args(**change):
    a = dict(q=torch.zeros(5, 128), out=torch.zeros(5, 128), kcache=torch.zeros(4, 1, 16, 64), vcache=torch.zeros(4, 1, 16, 64), block_tables=torch.zeros(2, 3, dtype=INT),
             seq_first_row=torch.zeros(3, dtype=INT), seq_start_pos=torch.zeros(2, dtype=INT), positions=torch.zeros(5, dtype=INT), visible=torch.zeros(5, 1, dtype=INT),
             max_rows_per_seq=3, nh=2, nkv=1, hd=64, page_size=16, scale=1.0, window=None, max_context=40, parts=None, status=torch.zeros(1, dtype=INT))
    a.update(change)
    return a


@pytest.mark.parametrize("change", [dict(q=torch.zeros(5, 127)), dict(out=torch.zeros(4, 128)), dict(q=torch.zeros(128, 5).T), dict(nh=3, q=torch.zeros(5, 192), out=torch.zeros(5, 192), nkv=2),
                                    dict(out=torch.zeros(5, 128, dtype=torch.bfloat16)), dict(kcache=torch.zeros(4, 1, 8, 64)), dict(vcache=torch.zeros(4, 1, 16, 32)),
                                    dict(vcache=torch.zeros(5, 1, 16, 64)), dict(kcache=torch.zeros(4, 1, 64, 16).transpose(2, 3)), dict(block_tables=torch.zeros(2, 3)),
                                    dict(block_tables=torch.zeros(6, dtype=INT)), dict(seq_first_row=torch.zeros(2, dtype=INT)), dict(seq_start_pos=torch.zeros(2)),
                                    dict(positions=torch.zeros(4, dtype=INT)), dict(visible=torch.zeros(5, dtype=INT)), dict(visible=torch.zeros(4, 1, dtype=INT)),
                                    dict(visible=torch.zeros(5, 1, dtype=torch.int64)), dict(max_rows_per_seq=1025), dict(window=0), dict(hd=0)])
def test_attention(change):
    with pytest.raises(kernels.KernelError):
        kernels.tree_attention(**attention_args(**change))


def test_attention_wants_the_gpu():
    with pytest.raises(kernels.KernelError, match="CUDA"):
        kernels.tree_attention(**attention_args())


def verify_args(**change):
    a = dict(logits=torch.zeros(5, 100), tokens=torch.zeros(5, dtype=INT), parents=torch.zeros(5, dtype=INT), seq_first_row=torch.zeros(3, dtype=INT), uniform=torch.zeros(5, 2),
             temperature=torch.zeros(2), path=torch.zeros(5, dtype=INT), accepted=torch.zeros(2, dtype=INT), next_token=torch.zeros(2, dtype=INT), draft_logits=None)
    a.update(change)
    return a


@pytest.mark.parametrize("change", [dict(logits=torch.zeros(100)), dict(logits=torch.zeros(100, 5).T), dict(logits=torch.zeros(5, 100, dtype=torch.float64)),
                                    dict(draft_logits=torch.zeros(5, 99)), dict(draft_logits=torch.zeros(5, 100, dtype=torch.bfloat16)), dict(tokens=torch.zeros(4, dtype=INT)),
                                    dict(parents=torch.zeros(5)), dict(seq_first_row=torch.zeros(2, dtype=INT)), dict(uniform=torch.zeros(5)), dict(uniform=torch.zeros(6, 2)),
                                    dict(uniform=torch.zeros(5, 2, dtype=torch.float64)), dict(temperature=torch.zeros(2, dtype=torch.float64)), dict(path=torch.zeros(4, dtype=INT)),
                                    dict(accepted=torch.zeros(1, dtype=INT)), dict(next_token=torch.zeros(2)), dict(logits=torch.zeros(5, 0))])
def test_verification(change):
    with pytest.raises(kernels.KernelError):
        kernels.verify_tree(**verify_args(**change))


def test_verification_of_a_vocabulary_that_is_too_large():
    big = torch.zeros(1, 1).expand(1, kernels.VERIFY_MAX_VOCAB + 1)
    with pytest.raises(kernels.KernelError):
        kernels.verify_tree(**verify_args(logits=big))


def keep_args(**change):
    a = dict(kpool=torch.zeros(2, 4, 1, 16, 64), vpool=torch.zeros(2, 4, 1, 16, 64), block_tables=torch.zeros(2, 3, dtype=INT), seq_first_row=torch.zeros(3, dtype=INT),
             seq_start_pos=torch.zeros(2, dtype=INT), path=torch.zeros(5, dtype=INT), accepted=torch.zeros(2, dtype=INT), page_size=16, max_rows_per_seq=3, status=torch.zeros(1, dtype=INT))
    a.update(change)
    return a


@pytest.mark.parametrize("change", [dict(kpool=torch.zeros(4, 1, 16, 64)), dict(vpool=torch.zeros(2, 4, 2, 16, 64)), dict(page_size=8), dict(kpool=torch.zeros(2, 4, 1, 16, 64, dtype=torch.uint8)),
                                    dict(block_tables=torch.zeros(2, 3)), dict(seq_first_row=torch.zeros(2, dtype=INT)), dict(path=torch.zeros(5)), dict(accepted=torch.zeros(1, dtype=INT)),
                                    dict(max_rows_per_seq=1025), dict(kpool=torch.zeros(2, 4, 1, 64, 16).transpose(3, 4))])
def test_keeping(change):
    with pytest.raises(kernels.KernelError):
        kernels.keep_rows(**keep_args(**change))


def test_keeping_wants_the_gpu():
    with pytest.raises(kernels.KernelError, match="CUDA"):
        kernels.keep_rows(**keep_args())
