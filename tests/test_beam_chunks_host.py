"""How far a beam search runs ahead of what it knows (no GPU needed)."""
import numpy as np
import pytest

from pvlc_b200 import beam


class Event:
    def __init__(self):
        self.waited = False

    def synchronize(self):
        self.waited = True


@pytest.mark.parametrize("steps", [0, 1, 3, 4, 5, 16, 17])
@pytest.mark.parametrize("chunk", [1, 4, 32])
def test_one_chunk_ahead(steps, chunk):
    """Requests that are done after any number of chunks (0: at their prompts, None: never): every
    step before that is queued, and one chunk at most behind it."""
    chunks = -(-steps // chunk)
    for end in [None, *range(chunks + 1)]:
        queued, events = [], []

        def status(n):
            # the flags are there once the event has been waited for
            events.append(Event())
            done = np.array([True, end is not None and n >= end])

            class Flags:
                def all(self, event=events[-1]):
                    assert event.waited
                    return done.all()
            return Flags(), events[-1]

        def queue(n):
            assert sum(e.waited for e in events) >= len(queued)      # one ahead, no more
            queued.append(n)
            return status(len(queued))
        beam.run_chunks(steps, chunk, status(0), queue)
        want = chunks if end is None else min(chunks, end + 1)
        assert len(queued) == want, (end, queued)
        assert queued == [min(chunk, steps - i * chunk) for i in range(want)]
        assert events[want if end is None else min(end, want)].waited
