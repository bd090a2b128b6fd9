"""A workload that reaches every kernel of the losses on logits, for the checked-build test (tests/test_gpu_losses_checked.py).

Run as `python tests/losses_workload.py OUT.npz` with MOTEOPT_LIB naming the library to load; writes every output to OUT.npz
and prints the library's index-check count (moteopt_check_count) on its last line.
"""

import sys
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent
sys.path.insert(0, str(ROOT))

import numpy as np  # noqa: E402
import torch  # noqa: E402


def main(out_path: str) -> None:
    import mote_b200 as m
    from mote_b200 import _lib as L
    dev = torch.device("cuda", 0)
    L.lib.moteopt_check_count(1)
    gen = torch.Generator(device=dev)
    gen.manual_seed(11)
    out = {}
    # one cluster and many blocks of tiles (8 lanes with 2, 5 and more lines, 32 lanes), slices of 128 and 256 threads and of
    # clusters, pieces of a stream; both types, shifted rows, ignored positions, targets that do not exist
    for dtype in (torch.bfloat16, torch.float32):
        for S, T, V in ((4, 9, 60), (4, 9, 271), (4, 7, 777), (4, 5, 2200), (8, 100, 271), (8, 100, 60), (6, 150, 900),
                        (6, 12, 4400), (4, 3, 9001), (2, 40, 30011), (2, 3, 140003), (4, 9000, 40)):
            name = f"{str(dtype)[6:]}_{S}_{T}_{V}_"
            z = (torch.randn(S, T + 1, V, generator=gen, device=dev) * 2).to(dtype)
            y = torch.randint(-3, V + 1, (S, T + 1), generator=gen, device=dev)
            y[0, 0] = V + 5
            for v, l, tag in ((z, y, "whole"), (z[:, :-1], y[:, 1:], "shifted")):
                r = m.token_logprobs(v, l, temperature=0.9)
                d = m.token_logprobs_backward(v, l, r.logprobs, r.lse, torch.ones_like(r.lse), temperature=0.9)
                w = (torch.arange(S, device=dev) % 3).float()
                p = m.policy_loss(v, l.clamp(max=V - 1), torch.randn(S, generator=gen, device=dev), r.logprobs.nan_to_num(),
                                  r.logprobs.nan_to_num(), weights=w, kl_coef=0.1, divisor=7.0)
                q = m.preference_loss(v, l.clamp(max=V - 1), average=True)
                flat = v.reshape(-1, V)
                cu = torch.linspace(1, flat.shape[0] - 1, S + 1, device=dev).to(torch.int32)
                k = m.preference_loss(flat, l.reshape(-1).clamp(max=V - 1), cu_seqlens=cu, label_smoothing=0.1)
                e = m.preference_loss(flat, l.reshape(-1).clamp(max=V - 1), cu_seqlens=cu, grad=False)
                for n, t in {"lp": r.logprobs, "lse": r.lse, "d": d, "pl": p.loss, "pk": p.kl, "pg": p.grad, "ql": q.loss,
                             "qg": q.grad, "kl": k.loss, "kg": k.grad, "el": e.loss}.items():
                    t = t.float().flatten()
                    out[name + tag + n] = t[:: max(1, t.numel() // 50000)].cpu().numpy()
    torch.cuda.synchronize()
    np.savez(out_path, **out)
    print("checks", L.lib.moteopt_check_count(1))


if __name__ == "__main__":
    main(sys.argv[1])
