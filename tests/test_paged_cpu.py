"""What the operators of paged serving refuse, and what they declare to write.  Refusals come before anything is looked for on a GPU."""
import pytest
import torch

from gpu_ipc_example_b200._ext import load

I, L, H, F = torch.int32, torch.int64, torch.float16, torch.float32


def ops():
    load()
    return torch.ops.b200ipc


def z(*shape, dtype=I):
    return torch.zeros(*shape, dtype=dtype)


def extend_args():
    return dict(block_table=z(3, 4), lens=z(3), new_lens=z(3), free_pages=z(9), n_free=z(1), page=16, rows=5)


def trim_args():
    return dict(block_table=z(3, 4), lens=z(3), keep_lens=z(3), free_pages=z(9), n_free=z(1), page=16)


def append_args():
    return dict(qkv=z(5, 4 * 128, dtype=H), kcache=z(3, 1, 16, 128, dtype=H), vcache=z(3, 1, 16, 128, dtype=H), slots=z(5, dtype=L), positions=z(5), hq=2, hkv=1,
                theta=1e4)


def attention_args():
    return dict(q=z(5, 2 * 128, dtype=H), kcache=z(3, 1, 16, 128, dtype=H), vcache=z(3, 1, 16, 128, dtype=H), block_table=z(3, 4), lens=z(3), cu_new=z(4),
                workspace=z(1 << 10, dtype=torch.uint8), hq=2, hkv=1, max_new=5)


def verify_args():
    return dict(target_probs=z(3, 5, 7, dtype=F), draft_probs=z(3, 4, 7, dtype=F), draft_tokens=z(3, 4, dtype=L), draft_lens=z(3), accept=z(3, 4, dtype=F),
                sample=z(3, dtype=F))


CASES = [
    ("paged_extend", extend_args, dict(block_table=z(3, 4, dtype=L)), "block table"),
    ("paged_extend", extend_args, dict(block_table=z(0, 4)), "block table"),
    ("paged_extend", extend_args, dict(block_table=z(4, 3).t()), "block table"),
    ("paged_extend", extend_args, dict(block_table=z(8193, 1), lens=z(8193), new_lens=z(8193)), "block table"),
    ("paged_extend", extend_args, dict(lens=z(4)), "lens"),
    ("paged_extend", extend_args, dict(new_lens=z(3, dtype=L)), "new_lens"),
    ("paged_extend", extend_args, dict(new_lens=z(6)[::2]), "new_lens"),
    ("paged_extend", extend_args, dict(free_pages=z(3, 3)), "free_pages"),
    ("paged_extend", extend_args, dict(n_free=z(2)), "n_free"),
    ("paged_extend", extend_args, dict(page=0), "page size"),
    ("paged_extend", extend_args, dict(rows=-1), "rows"),
    ("paged_extend", extend_args, dict(), "CUDA device"),
    ("paged_trim", trim_args, dict(block_table=z(3)), "block table"),
    ("paged_trim", trim_args, dict(keep_lens=z(2)), "keep_lens"),
    ("paged_trim", trim_args, dict(free_pages=z(9, dtype=L)), "free_pages"),
    ("paged_trim", trim_args, dict(page=-1), "page size"),
    ("paged_trim", trim_args, dict(), "CUDA device"),
    ("rope_paged_append", append_args, dict(qkv=z(5, 4 * 128, dtype=F)), "float16 and bfloat16"),
    ("rope_paged_append", append_args, dict(qkv=z(5, 3 * 128, dtype=H)), "rows of at least"),
    ("rope_paged_append", append_args, dict(qkv=z(4 * 128, 5, dtype=H).t()), "rows of at least"),
    ("rope_paged_append", append_args, dict(qkv=z(5, 4 * 128 + 4, dtype=H)[:, :512]), "16-byte"),
    ("rope_paged_append", append_args, dict(kcache=z(3, 1, 16, 64, dtype=H), vcache=z(3, 1, 16, 64, dtype=H)), "caches"),
    ("rope_paged_append", append_args, dict(kcache=z(3, 1, 16, 128, dtype=torch.bfloat16)), "caches"),
    ("rope_paged_append", append_args, dict(vcache=z(3, 1, 32, 128, dtype=H)), "caches"),
    ("rope_paged_append", append_args, dict(kcache=z(0, 1, 16, 128, dtype=H), vcache=z(0, 1, 16, 128, dtype=H)), "no pages"),
    ("rope_paged_append", append_args, dict(hq=3, hkv=2), "multiple"),
    ("rope_paged_append", append_args, dict(slots=z(5)), "slots"),
    ("rope_paged_append", append_args, dict(positions=z(4)), "positions"),
    ("rope_paged_append", append_args, dict(theta=0.0), "theta"),
    ("rope_paged_append", append_args, dict(theta=float("inf")), "theta"),
    ("rope_paged_append", append_args, dict(), "CUDA device"),
    ("paged_attention", attention_args, dict(q=z(5, 128, dtype=H)), "rows of at least"),
    ("paged_attention", attention_args, dict(q=z(5, 256 + 4, dtype=H)[:, 4:]), "16-byte"),
    ("paged_attention", attention_args, dict(kcache=z(3, 1, 24, 128, dtype=H), vcache=z(3, 1, 24, 128, dtype=H)), "pages of 16"),
    ("paged_attention", attention_args, dict(block_table=z(3, 4, dtype=L)), "block table"),
    ("paged_attention", attention_args, dict(block_table=z(1, 1 << 27), lens=z(1), cu_new=z(2)), "2.30 positions"),
    ("paged_attention", attention_args, dict(q=z(1, 8192 * 128, dtype=H), kcache=z(1, 8192, 16, 128, dtype=H), vcache=z(1, 8192, 16, 128, dtype=H),
                                             block_table=torch.empty(8, 1 << 22, dtype=I), lens=z(8), cu_new=z(9), hq=8192, hkv=8192), "2.42 in the whole table"),
    ("paged_attention", attention_args, dict(cu_new=z(3)), "cu_new"),
    ("paged_attention", attention_args, dict(lens=z(3, dtype=L)), "lens"),
    ("paged_attention", attention_args, dict(max_new=0), "max_new"),
    ("paged_attention", attention_args, dict(q=z(5, 65 * 128, dtype=H), hq=65), "64 query heads"),
    ("paged_attention", attention_args, dict(), "CUDA device"),
    ("verify_drafts", verify_args, dict(draft_tokens=z(3, 4)), "draft_tokens"),
    ("verify_drafts", verify_args, dict(draft_tokens=z(3, dtype=L)), "draft_tokens"),
    ("verify_drafts", verify_args, dict(accept=z(3, 5, dtype=F)), "accept"),
    ("verify_drafts", verify_args, dict(sample=z(3, dtype=torch.float64)), "sample"),
    ("verify_drafts", verify_args, dict(draft_lens=z(3, dtype=L)), "draft_lens"),
    ("verify_drafts", verify_args, dict(target_probs=z(3, 4, 7, dtype=F)), "target_probs"),
    ("verify_drafts", verify_args, dict(target_probs=z(3, 5, 7, dtype=H)), "target_probs"),
    ("verify_drafts", verify_args, dict(target_probs=z(3, 5, 14, dtype=F)[..., ::2]), "target_probs"),
    ("verify_drafts", verify_args, dict(target_probs=z(3, 5, 0, dtype=F), draft_probs=None), "target_probs"),
    ("verify_drafts", verify_args, dict(draft_probs=z(3, 4, 8, dtype=F)), "draft_probs"),
    ("verify_drafts", verify_args, dict(), "CUDA device"),
]


@pytest.mark.parametrize("name,args,change,message", CASES, ids=[f"{c[0]}-{'-'.join(c[2]) or 'cpu'}-{i}" for i, c in enumerate(CASES)])
def test_refusals(name, args, change, message):
    with pytest.raises(RuntimeError, match=message):
        getattr(ops(), name)(**{**args(), **change})


@pytest.mark.parametrize("name,written", [
    ("paged_extend", {"block_table", "lens", "n_free"}),
    ("paged_trim", {"block_table", "lens", "free_pages", "n_free"}),
    ("rope_paged_append", {"kcache", "vcache"}),
    ("paged_attention", {"workspace"}),
    ("verify_drafts", set()),
])
def test_written_arguments_are_declared(name, written):
    schema = getattr(ops(), name).default._schema
    assert {a.name for a in schema.arguments if a.alias_info is not None and a.alias_info.is_write} == written
