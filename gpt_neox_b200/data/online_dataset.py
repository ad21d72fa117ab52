"""Dataset fed by an online sampling server (REINFORCE-style training,
``megatron/data/online_dataset.py:29-128``): each request returns a pickled
``{"prefix": [...], "completions": [[...], ...], "rewards": [...]}`` batch; rewards are centred with a
leave-one-out baseline or a moving average, and every completion becomes one sample with the prompt positions
labelled -100.  An optional ``"logprobs": [[...], ...]`` (of every completion's tokens under the policy that sampled them) becomes
``old_logp``, which ``reinforce_clip`` needs (``needs_logprobs``: a batch without them is an error)."""
from __future__ import annotations

import pickle
import socket
import time
from collections import deque

import numpy as np
import torch


class OnlineDataset(torch.utils.data.Dataset):
    def __init__(self, num_samples, seq_length, leave_one_out=False, data_split="train", dataserver_ips="localhost",
                 dataserver_ports=10000, needs_logprobs=False):
        self.num_samples, self.seq_length, self.leave_one_out = num_samples, seq_length, leave_one_out
        self.data_split, self.needs_logprobs = data_split, needs_logprobs
        self.ips = dataserver_ips if isinstance(dataserver_ips, (list, tuple)) else [dataserver_ips]
        self.ports = dataserver_ports if isinstance(dataserver_ports, (list, tuple)) else [dataserver_ports]
        self.queue = deque()
        self.reward_window = deque(maxlen=100)
        self._rr = 0

    def __len__(self):
        return self.num_samples

    def _fetch(self):
        ip = self.ips[self._rr % len(self.ips)]
        port = self.ports[self._rr % len(self.ports)]
        self._rr += 1
        while True:
            try:
                with socket.create_connection((ip, port), timeout=60) as s:
                    s.sendall(self.data_split.encode())
                    buf = b""
                    while True:
                        chunk = s.recv(1 << 20)
                        if not chunk:
                            break
                        buf += chunk
                return pickle.loads(buf)
            except (ConnectionRefusedError, socket.timeout):
                time.sleep(1.0)

    def _fill(self):
        batch = self._fetch()
        rewards = np.asarray(batch["rewards"], dtype=np.float32)
        if self.leave_one_out and len(rewards) > 1:
            baseline = (rewards.sum() - rewards) / (len(rewards) - 1)
        else:
            self.reward_window.extend(rewards.tolist())
            baseline = np.full_like(rewards, float(np.mean(self.reward_window)))
        centred = rewards - baseline
        prefix = list(batch["prefix"])
        # log-probabilities of the completions' tokens under the policy that sampled them, for the clipped loss
        logps = batch.get("logprobs")
        if logps is None or len(logps) == 0:
            if self.needs_logprobs:
                raise ValueError("reinforce_clip compares with the sampler's log-probabilities, and the data server sent no logprobs")
            logps = [None] * len(batch["completions"])
        elif len(logps) != len(batch["completions"]):
            raise ValueError(f"the data server sent log-probabilities of {len(logps)} completions with {len(batch['completions'])}")
        for comp, rw, raw, logp in zip(batch["completions"], centred, rewards, logps):
            toks = (prefix + list(comp))[: self.seq_length + 1]
            n = len(toks)
            text = np.zeros(self.seq_length + 1, dtype=np.int64)
            text[:n] = toks
            label = np.full(self.seq_length + 1, -100, dtype=np.int64)
            label[len(prefix):n] = toks[len(prefix):n]
            sample = {"text": text, "label": label, "reward": np.full(self.seq_length + 1, rw, np.float32),
                      "raw_reward": np.float32(raw)}
            if logp is not None:
                if len(logp) != len(comp):
                    raise ValueError(f"the data server sent {len(logp)} log-probabilities for {len(comp)} tokens")
                old = np.zeros(self.seq_length + 1, dtype=np.float32)
                old[len(prefix):n] = np.asarray(logp, dtype=np.float32)[: max(n - len(prefix), 0)]
                sample["old_logp"] = old
            self.queue.append(sample)

    def __getitem__(self, idx):
        while not self.queue:
            self._fill()
        return self.queue.popleft()
