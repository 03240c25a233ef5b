"""Two EP buffers of one process whose traffic goes through their proxies at
the same time: their copy lanes share streams. Spawned with RANK/WORLD_SIZE."""

from __future__ import annotations

import os
import signal

signal.alarm(100)

import torch
import torch.distributed as dist

T, H, K, ROUNDS = 96, 256, 2, 3


def inputs(rank, which, turn, experts):
    g = torch.Generator().manual_seed(1000 * rank + 10 * which + turn)
    x = torch.randn(T, H, generator=g).bfloat16()
    idx = torch.rand(T, experts, generator=g).argsort(-1)[:, :K].contiguous()
    return x, idx, torch.rand(T, K, generator=g)


def main():
    rank, world = int(os.environ["RANK"]), int(os.environ["WORLD_SIZE"])
    dist.init_process_group("gloo", rank=rank, world_size=world)
    torch.cuda.set_device(0)
    import uccl_amd.ep as ep

    experts = 4 * world
    bufs = [ep.Buffer(num_experts=experts, topk=K, hidden=H, max_tokens=128)
            for _ in range(2)]
    for turn in range(ROUNDS):
        own = [inputs(rank, b, turn, experts) for b in range(2)]
        on_gpu = [[t.cuda() for t in o] for o in own]
        for b, buf in enumerate(bufs):
            buf.dispatch_send(on_gpu[b][0], on_gpu[b][1])
        for buf in bufs:
            buf.dispatch_recv()
        outs = [buf.recv_x_view() * 2 for buf in bufs]
        for b, buf in enumerate(bufs):
            buf.combine_send(outs[b])
        got = [buf.combine_recv(on_gpu[b][1], on_gpu[b][2])
               for b, buf in enumerate(bufs)]
        torch.cuda.synchronize()
        for b, buf in enumerate(bufs):
            buf._b.check_error()
            x, _, w = own[b]
            want = x.double() * 2 * w.double().sum(-1, keepdim=True)
            # K terms in 32 bits, rounded to bfloat16
            tol = want.abs() * (2.0 ** -8 + 4 * 2.0 ** -23)
            assert ((got[b].cpu().double() - want).abs() <= tol).all(), (turn, b)
        print(f"[rank {rank}] round {turn} OK", flush=True)
    dist.barrier()
    for buf in bufs:
        buf.close()
    print("TWO BUFFERS OK", flush=True)
    dist.destroy_process_group()


if __name__ == "__main__":
    main()
