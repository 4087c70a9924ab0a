"""The error word of the dense operators, with checks on several streams at once."""
import threading

import pytest
import torch

import apoe

pytestmark = pytest.mark.gpu


def test_every_raised_error_is_reported_exactly_once():
    """Checks that run at the same time on several streams: what one of them has reported no other reports again, and an error
    raised while another stream is checked is not lost."""
    raises, found, done = 300, [], threading.Event()

    def look(stream):
        try:
            apoe.dense_check_status(0, apoe.C.c_void_p(stream.cuda_stream))
        except apoe.ApoeError as e:
            assert e.code == 6
            found.append(1)

    def others():
        stream = torch.cuda.Stream()
        while not done.is_set():
            look(stream)

    apoe.dense_check_status()
    threads = [threading.Thread(target=others) for _ in range(2)]
    for t in threads:
        t.start()
    stream = torch.cuda.Stream()
    for _ in range(raises):
        apoe._check(apoe.lib().ap_debug_dense_wait_timeout(0, 1, apoe.C.c_void_p(stream.cuda_stream)))
        stream.synchronize()
        look(stream)                                  # this check or one of the others: after it nothing is left
    done.set()
    for t in threads:
        t.join()
    assert len(found) == raises
    apoe.dense_check_status()
