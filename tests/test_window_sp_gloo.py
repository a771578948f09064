"""The block's windowed attention under sequence parallelism: two CPU ranks (gloo) with uneven shares of the
tokens get the rows of the whole sequence's attention, positions and first tokens counted over the
whole sequence.  The kernel is stood in for by its plain form."""
import os
import socket
import sys
from pathlib import Path

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

ROOT = Path(__file__).resolve().parents[1]


def _worker(rank, world, port, seq, heads, window, sinks, result_dir):
    sys.path[:0] = [str(ROOT), str(ROOT / "tests")]
    import importlib

    import operator_refs as R
    os.environ["MASTER_ADDR"] = "127.0.0.1"
    os.environ["MASTER_PORT"] = str(port)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        pkg = importlib.import_module("dcu-video-dit-turbo_b200")
        from oracle import ref_ops as ref
        calls = []

        def plain(q, k, v, scale, left, right, first=0, lengths=None):
            calls.append((left, right, first, q.shape[1]))
            assert q.shape[2] == seq                        # the whole sequence, a share of the heads
            out = R.window_attention(q, k, v, scale, left, right, first).to(torch.bfloat16)
            return out.transpose(1, 2).contiguous().transpose(1, 2)

        pkg.block.ops.window_fwd_bhsd = plain
        D = 16
        splits = pkg.ulysses.sequence_splits(seq, world)
        sp = pkg.ulysses.UlyssesSP(splits, heads, D)
        g = torch.Generator().manual_seed(7)
        qkv = torch.randn((seq, 3, heads, D), generator=g).to(torch.bfloat16)
        start = sum(splits[:rank])
        mine = qkv[start:start + splits[rank]].contiguous()
        params = {"heads": heads, "head_dim": D, "ffn": 64}
        q, k, v = (qkv[:, i].transpose(0, 1).unsqueeze(0) for i in range(3))
        whole = plain(q, k, v, D ** -0.5, *window, sinks)[0].transpose(0, 1).reshape(seq, heads * D)
        want = whole[start:start + splits[rank]]
        for chunks in (1, heads // world):
            block = pkg.block.DiTBlock(params, sp=sp, head_chunks=chunks, overlap=False, fuse_swiglu=False, window=window, sinks=sinks)
            calls.clear()
            assert torch.equal(block.attention(mine), want)
            assert calls == [(*window, sinks, heads // world // chunks)] * chunks
            gathered = sp.attention_packed(ref.pack_send(mine, world, chunks), block._attn, overlap=False)
            assert torch.equal(sp.unpack_gathered(gathered), want)
        Path(result_dir, f"r{rank}.txt").write_text("ok")
    finally:
        dist.destroy_process_group()


@pytest.mark.parametrize("seq,heads,window,sinks", [(23, 4, (5, 0), 2), (30, 6, (4, 7), 3), (31, 2, (-1, 0), 0)])
def test_windowed_block_on_two_ranks(tmp_path, seq, heads, window, sinks):
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    mp.spawn(_worker, args=(2, port, seq, heads, window, sinks, str(tmp_path)), nprocs=2, join=True)
    assert [Path(tmp_path, f"r{r}.txt").read_text() for r in range(2)] == ["ok", "ok"]
