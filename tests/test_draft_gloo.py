"""Drafted tokens through a tensor-parallel decoder on CPU: two gloo ranks, with plain tensor operations in place of the CUDA library (the
wiring, the shards and the exchange are what is under test)."""
import os
import socket

import numpy as np
import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp


def _free_port():
    s = socket.socket()
    s.bind(("127.0.0.1", 0))
    p = s.getsockname()[1]
    s.close()
    return p


def _stand_ins(C):
    """The entry points of flh_b200._CUDA that a drafted pass calls, on CPU tensors."""
    from oracle import oracle as O

    def act_quant_group(x, group, hadamard):
        q, s = O.quant_group_sym(np.ascontiguousarray(x.reshape(-1, 128).numpy()), hadamard)
        return torch.from_numpy(q.copy()).view(x.shape[:-1] + (x.shape[-1] // 2,)), torch.from_numpy(s.copy()).view(x.shape[:-1] + (x.shape[-1] // 128,))

    def act_quant_token(x, hadamard, clip):
        q, s, z = O.quant_token_asym(np.ascontiguousarray(x.reshape(-1, x.shape[-1]).numpy()), hadamard, clip)
        lead = x.shape[:-1]
        return torch.from_numpy(q.copy()).view(lead + (x.shape[-1] // 2,)), torch.from_numpy(s.copy()).view(lead + (1,)), torch.from_numpy(z.copy()).view(lead + (1,))

    def gemm(A, B, A_scale, B_scale, A_zero=None, B_rowsum=None, bias=None, out_dtype=torch.float16, algo=0, out=None):
        return torch.from_numpy(O.gemm_i4_dequant(A.numpy(), B.numpy(), A_scale.numpy(), B_scale.numpy(), a_zero=None if A_zero is None else A_zero.numpy()).copy())

    def rope_kv_at(qkv, cos, sin, positions, lengths, k, v, nh):
        B, S = positions.shape
        nkv, D = k.shape[1], k.shape[3]
        x = qkv.view(B, S, nh + 2 * nkv, D)
        c, s = cos[positions.long()][:, :, None], sin[positions.long()][:, :, None]
        x1, x2 = x[:, :, :nh + nkv, :D // 2].float(), x[:, :, :nh + nkv, D // 2:].float()
        turned = torch.cat((x1 * c - x2 * s, x2 * c + x1 * s), dim=-1).half()
        for b, n in enumerate(lengths.tolist()):
            k[b, :, n:n + S], v[b, :, n:n + S] = turned[b, :, nh:].transpose(0, 1), x[b, :, nh + nkv:].transpose(0, 1)
        return turned[:, :, :nh].contiguous()

    def tree_attention(q, k, v, lengths, tree=None, weights=None, scale=None, counted=None):
        out = torch.empty_like(q)
        B, S, nh, D = q.shape
        g = nh // k.shape[1]
        for b, n in enumerate(lengths.tolist()):
            seen = torch.ones(S, n + S, dtype=torch.bool)
            seen[:, n:] = torch.ones(S, S).tril().bool() if tree is None else torch.tensor([[bool((int(t) >> j) & 1) for j in range(S)] for t in tree])
            for h in range(nh):
                p = (q[b, :, h].double() @ k[b, h // g, :n + S].double().t() / D ** 0.5).masked_fill(~seen, -torch.inf).softmax(-1)
                out[b, :, h] = (p @ v[b, h // g, :n + S].double()).half()
                if weights is not None:
                    weights[b, h // g, :n + S] += p[:S if counted is None else int(counted[b])].sum(0)
        return out

    def cache_accept(ks, vs, lengths, path, accepted, drafted, weights=None):
        for i, (k, v) in enumerate(zip(ks, vs)):
            for b, (n, a) in enumerate(zip(lengths.tolist(), accepted.tolist())):
                at = [n + int(j) for j in path[b, :a]]
                k[b, :, n:n + a], v[b, :, n:n + a] = k[b][:, at], v[b][:, at]
                if weights is not None:
                    weights[i][b, :, n:n + a] = weights[i][b][:, at]
                    weights[i][b, :, n + a:n + drafted] = 0
        return lengths + accepted

    def sdpa(q, k, v, attn_mask=None, is_causal=False, enable_gqa=False):
        g = q.shape[1] // k.shape[1]
        x = q.double() @ k.double().repeat_interleave(g, 1).transpose(-1, -2) / q.shape[-1] ** 0.5
        x = x.masked_fill(~torch.ones(x.shape[-2:], dtype=torch.bool).tril(), -torch.inf) if is_causal else x
        return (x.softmax(-1) @ v.double().repeat_interleave(g, 1)).half()

    # both attentions in 64 bits: rounded to 16 they agree, and so does everything behind them
    torch.nn.functional.scaled_dot_product_attention = sdpa
    for f in (act_quant_group, act_quant_token, rope_kv_at, tree_attention, cache_accept):
        setattr(C, f.__name__, f)
    C.gemm_i4_dequant = gemm
    C.weight_rowsum = lambda B, group: torch.from_numpy(O.weight_rowsum(B.numpy(), group))
    C.square_f32 = lambda x: None


def _worker(rank, world, port, tmp, mode):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    torch.set_num_threads(2)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        import flh_b200
        from flh_b200.draft import DraftTree
        from flh_b200.model import Decoder, DecoderConfig, rope_tables
        _stand_ins(flh_b200._CUDA)
        cfg = DecoderConfig(hidden=256, n_heads=4, n_kv_heads=2, ffn=512, n_layers=2, vocab=64, act_mode=mode, tp=world, max_positions=64, seq_parallel=False,
                            fuse_glue=False)       # forward() and the MLP as tensor operations
        m = Decoder(cfg, torch.device("cpu"), seed=3)
        m._tables[64] = rope_tables(torch.arange(64), cfg.head_dim, cfg.rope_theta)          # (made and waited for on a device otherwise)
        gen = torch.Generator().manual_seed(5)
        prompt, ids, tree = torch.randint(0, 64, (2, 9), generator=gen), torch.randint(0, 64, (2, 5), generator=gen), DraftTree([-1, 0, 0, 1, 3])
        whole = {i: m(torch.cat((prompt, ids[:, [j for j in range(5) if (int(tree.bits[i]) >> j) & 1]]), dim=1)) for i in range(5)}
        for observe in (False, True):
            cache, lengths = m.new_cache(2, 40, observe=observe), torch.zeros(2, dtype=torch.int32)
            for i in range(9):                           # the prompt, one token at a time
                m.draft(prompt[:, i:i + 1], cache, lengths)
                lengths = lengths + 1
            logits = m.draft(ids, cache, lengths, tree)
            every = [torch.empty_like(logits) for _ in range(world)]
            dist.all_gather(every, logits)
            assert all(torch.equal(x, logits) for x in every), "the ranks' logits"
            for i in range(5):
                assert torch.equal(logits[:, i:i + 1], whole[i][:, -1:]), i
            now = m.accept(cache, lengths, torch.tensor([[0, 1, 3], [0, 2, 0]], dtype=torch.int32), torch.tensor([3, 2], dtype=torch.int32), 5)
            assert now.tolist() == [12, 11]
            for c in cache if observe else ():
                assert torch.allclose(c[3].sum(-1), torch.tensor([[12.0 * 2], [11.0 * 2]]), rtol=1e-3) and not c[3][1, :, 11:].any()
        if rank == 0:
            open(os.path.join(tmp, "ok"), "w").write("ok")
    finally:
        dist.destroy_process_group()


@pytest.mark.parametrize("mode", ["group_sym", "token_asym"])
def test_drafts_of_a_tensor_parallel_decoder(tmp_path, mode):
    mp.spawn(_worker, args=(2, _free_port(), str(tmp_path), mode), nprocs=2, join=True)
    assert (tmp_path / "ok").exists()
