// stream_order.hpp -- what a call of a context has to wait for on the GPU.
//
// A call may leave work behind on its stream that uses the context's scratch, or memory that the next call gives back, and the next call may run on another
// stream.  One event stands for all that work: the call's own stream is put behind it before anything of the call is launched, so that an event recorded there
// later covers both.  A stream that is being captured into a graph takes no part: an event from outside may not be waited for there, nor one from inside outside.  It
// owes the wait, and the first call that finds it no longer captured pays.
//
// Api: lasting(s): the stream will not be destroyed by the caller; captured(s); record(s) and wait(s): the event's.  (A fake of it in the tests stands for a GPU.)
#pragma once

namespace vqb {

template <typename Api> class StreamOrder {
    using Stream = typename Api::Stream;
    bool unfinished_ = false; // nothing has waited for the calls' work since the last launch or copy
    bool owed_ = false;       // the present stream is not behind the event yet
    bool late_ = false;       // nor the event behind `from_`, on which nothing could be recorded (the default stream while another one is being captured)
    Stream from_{};

  public:
    Api api;

    void launched() { unfinished_ = true; }
    // The host has waited for the present stream.
    void waited()
    {
        if (!owed_) unfinished_ = false;
    }

    // The caller may destroy a stream of its own as soon as its work is done, so such a stream gets the event while the call is still there (call_ends); a lasting
    // one gets it here, so that programs that never change streams pay nothing.
    void change(Stream old, Stream now)
    {
        if (old == now || !unfinished_) return;
        if (api.lasting(old) && (!owed_ || late_)) {
            if (api.captured(old)) late_ = true, from_ = old;
            else api.record(old);
        }
        owed_ = true;
        settle(now);
    }

    // Before a call launches or gives back anything.
    void settle(Stream now)
    {
        if (!owed_ || api.captured(now)) return;
        api.wait(now);
        if (late_) {
            if (api.captured(from_)) return;
            api.record(from_);
            api.wait(now);
            late_ = false;
        }
        owed_ = false;
    }

    void call_ends(Stream now)
    {
        if (!unfinished_ || api.lasting(now) || api.captured(now)) return;
        settle(now); // (a capture may have ended meanwhile)
        api.record(now);
    }
};

} // namespace vqb
