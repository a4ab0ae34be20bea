// The paged attention's schedule (paged_sched.h) as a host library, for tests/test_paged_sched.py.
#include "../rosylnalive_b200/csrc/paged_sched.h"

using namespace lrm::sched;

extern "C" {

int ring_stages() { return kRing; }
int lead_of(int wide) { return wide ? kLeadWide : kLead; }
int place_of_k(int t, int lead) { return k_place(t, lead); }
int place_of_v(int t, int nt, int lead) { return v_place(t, nt, lead); }
int marks() { return kMarks; }
int issuer_waits() { return (int)kIssuerWaits; }
int polls(int softmax) { return (int)(softmax ? kSoftmaxPolls : kPolls); }
int parity_of(int x) { return (int)fill_parity(x); }

}  // extern "C"
